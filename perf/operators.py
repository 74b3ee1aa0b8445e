"""The language-model operators that performance is measured on: a key/value cache held in 4 or 8 bits.

  store   new rows of keys and values are quantised into the cache's pages and read back from there
  read    rows that lie in the cache are read back
  attend  queries attend to the cache of their sequences: single tokens, a few tokens, prompts; all earlier tokens
          visible, or a sliding window and a few first tokens

A row is the D numbers of one token and one head.  It is held as integers c of 0..L, L = 2^bits - 1, with an offset m and a step s
in bfloat16: m is the largest bfloat16 that is not above the row's minimum, s the smallest that is not below
(maximum - m) / L, c = rint((x - m) / s), and it stands for m + s c.

`own` chooses between the framework's operators and their plain form in torch, in 32 bits."""
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEVICE = "cuda"
_context = None


# ---- cases -----------------------------------------------------------------------------------------------------------
def _store(name, seqs, tokens, heads, dim, bits, dtype, start=0, fused=False, page=64):
    """`seqs` sequences of about `tokens` new tokens, written from position `start` on; fused: keys and values are parts of rows
    that hold queries too"""
    return dict(name=name, kind="store", seqs=seqs, tokens=tokens, heads=heads, dim=dim, bits=bits, dtype=dtype, start=start,
                fused=fused, page=page)


def _read(name, seqs, tokens, heads, dim, bits, dtype, page=64):
    return dict(name=name, kind="read", seqs=seqs, tokens=tokens, heads=heads, dim=dim, bits=bits, dtype=dtype, page=page)


def _attend(name, seqs, kv_min, kv_max, q_min, q_max, heads, kv_heads, dim, bits, dtype, window=0, sinks=0, page=64):
    """lengths of the sequences are spread over kv_min..kv_max, their numbers of queries over q_min..q_max"""
    return dict(name=name, kind="attend", seqs=seqs, kv_min=kv_min, kv_max=kv_max, q_min=q_min, q_max=q_max, heads=heads,
                kv_heads=kv_heads, dim=dim, bits=bits, dtype=dtype, window=window, sinks=sinks, page=page)


def listed():
    return [
        # one new token of each sequence of a small batch: what every step of generation adds (latency)
        _store("store_step", 16, 1, 8, 128, 4, "bf16", start=777),
        # a long prompt of one sequence
        _store("store_prompt", 1, 8199, 8, 128, 4, "bf16"),
        # prompts of different lengths in one batch, float32, keys and values beside the queries in one tensor, an odd head size
        _store("store_ragged", 5, 700, 5, 80, 8, "f32", start=37, fused=True, page=32),
        # one sequence's rows for another program (moved, scored, cached elsewhere)
        _read("read_short", 1, 777, 2, 64, 4, "f16", page=32),
        # a batch of long sequences is taken out of the cache
        _read("read_long", 4, 16384, 8, 128, 4, "bf16"),
        # one user's next token, the smallest step (latency)
        _attend("step_one", 1, 513, 513, 1, 1, 32, 8, 128, 4, "bf16"),
        # a batch's next tokens, contexts of all lengths
        _attend("step_batch", 64, 61, 8192, 1, 1, 32, 8, 128, 4, "bf16"),
        # one long document's next token
        _attend("step_long", 1, 131072, 131072, 1, 1, 64, 8, 128, 4, "bf16"),
        # next tokens of models with windows and first tokens that stay visible; no shared heads
        _attend("step_window", 32, 3000, 40000, 1, 1, 16, 16, 64, 4, "f16", window=2048, sinks=4),
        # a few tokens at once (a draft to be checked), an odd head size, 8 bits
        _attend("draft", 24, 100, 5000, 3, 7, 20, 5, 80, 8, "bf16", page=32),
        # a prompt, each token seeing those before it
        _attend("prompt", 1, 8192, 8192, 8192, 8192, 32, 8, 128, 4, "bf16"),
        # parts of prompts behind what is already there, with a window
        _attend("chunk_window", 3, 4000, 16000, 300, 1000, 16, 4, 128, 4, "bf16", window=1024, sinks=16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("store", "read", "attend", "attend", "attend"))
    dim = rng.choice((64, 128, 128, rng.randrange(8, 257)))
    bits, dtype, page = rng.choice((4, 4, 8)), rng.choice(("bf16", "bf16", "f16")), rng.choice((32, 64, 128))
    kv_heads = rng.choice((1, 2, 3, 4, 5, 8, 16))
    if kind == "store":
        case = _store("", _log(rng, 1, 64), _log(rng, 1, 8000), kv_heads, dim, bits, rng.choice(("bf16", "f16", "f32")),
                      start=rng.choice((0, rng.randrange(3000))), fused=rng.random() < 0.4, page=page)
    elif kind == "read":
        case = _read("", _log(rng, 1, 64), _log(rng, 3, 16000), kv_heads, dim, bits, rng.choice(("bf16", "f16", "f32")), page=page)
    else:
        form = rng.choice(("step", "few", "prompt"))
        hi = _log(rng, 33, 100000 if form == "step" else 12000)
        q = 1 if form == "step" else _log(rng, 2, 16) if form == "few" else _log(rng, 17, 4000)
        hi = max(hi, q)
        lo = max(q, _log(rng, 1, hi))
        window = rng.choice((0, 0, _log(rng, 16, 4096)))
        case = _attend("", _log(rng, 1, 64), lo, hi, max(1, q - rng.randrange(1 + q // 2)), q, kv_heads * rng.choice((1, 2, 4, 7, 8)), kv_heads,
                       dim, bits, dtype, window=window, sinks=rng.choice((0, 1, 4, 33)) if window else 0, page=page)
    del case["name"]
    top = {"store": "store_prompt", "read": "read_long", "attend": "prompt"}
    limit = {k: work(next(c for c in listed() if c["name"] == n)) for k, n in top.items()}[kind]
    while _cost(case) > (limit["flops"] if kind == "attend" else limit["bytes"]):   # no more than the largest listed one
        if case["seqs"] > 1:
            case["seqs"] = (case["seqs"] + 1) // 2
        elif kind == "attend":
            for k in ("kv_min", "kv_max", "q_min", "q_max"):
                case[k] = (case[k] + 1) // 2
        else:
            case["tokens"] = (case["tokens"] + 1) // 2
    return case


def _cost(case):
    """what draw() bounds: bytes, or for attention the operations, a byte counted as 1900 of them (the largest listed batch and the
    largest prompt come to the same)"""
    w = work(case)
    return max(w["flops"], 1900 * w["bytes"]) if case["kind"] == "attend" else w["bytes"]


def _spread(lo, hi, n, salt):
    """n lengths of lo..hi, both of them among these, in an order of no meaning"""
    v = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(salt).shuffle(v)
    return v


def _lengths(case):
    """(tokens in the cache, new tokens or queries) of each sequence"""
    n = case["seqs"]
    if case["kind"] == "store":
        q = _spread(max(1, case["tokens"] // 2), case["tokens"], n, 1)
        return [case["start"] + v for v in q], q
    if case["kind"] == "read":
        kv = _spread(max(1, case["tokens"] // 2), case["tokens"], n, 1)
        return kv, kv
    q = _spread(case["q_min"], case["q_max"], n, 2)
    return [max(a, b) for a, b in zip(_spread(case["kv_min"], case["kv_max"], n, 3), q)], q


def work(case):
    kv, q = _lengths(case)
    bits, dim, dtype = case["bits"], case["dim"], TYPES[case["dtype"]]
    held = 2 * (dim * bits / 8 + 4)                  # a token's two rows of one head in the cache
    if case["kind"] != "attend":
        rows = sum(q) * case["heads"]
        out = rows * (2 * dim * dtype.itemsize + held)
        return {"bytes": 2 * out if case["kind"] == "store" else out, "flops": rows * dim * (16 if case["kind"] == "store" else 4)}
    window, sinks = case["window"], case["sinks"]
    pairs = tokens = 0
    for n, k in zip(kv, q):
        first = n - k                                # the position of the first query
        if not window:
            pairs += k * first + k * (k + 1) // 2
            tokens += n
        else:
            pairs += sum(min(p + 1, window + min(sinks, max(0, p + 1 - window))) for p in range(first, n))
            low = max(0, first + 1 - window)
            tokens += n - low + min(sinks, low)
    rows = sum(q) * case["heads"]
    return {"bytes": tokens * case["kv_heads"] * held + 2 * rows * dim * dtype.itemsize, "flops": 4 * dim * case["heads"] * pairs}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _rows(gen, tokens, heads, dim, dtype):
    """keys or values as layers produce them: channels of different size and offset, some of them far larger than the rest"""
    size = torch.rand(heads, dim, generator=gen, device=DEVICE) * 1.5 + 0.25
    shift = torch.randn(heads, dim, generator=gen, device=DEVICE) * (torch.rand(heads, dim, generator=gen, device=DEVICE) < 0.05) * 4
    x = torch.empty(tokens, heads, dim, dtype=dtype, device=DEVICE)
    for a in range(0, tokens, 1 << 16):
        b = min(tokens, a + (1 << 16))
        x[a:b] = torch.randn(b - a, heads, dim, generator=gen, device=DEVICE) * size + shift
    return x


def _layout(case, gen):
    """pages of the sequences in an order of no meaning: (page table [seqs, most], slots of all tokens, sequence by sequence)"""
    kv, _ = _lengths(case)
    page = case["page"]
    need = [-(-n // page) for n in kv]
    order = torch.randperm(sum(need) + 2, generator=gen, device=DEVICE)[:sum(need)].to(torch.int32)   # two pages stay unused
    table = torch.zeros(len(kv), max(need), dtype=torch.int32, device=DEVICE)
    at, slots = 0, []
    for i, n in enumerate(kv):
        own_pages = order[at:at + need[i]]
        table[i, :need[i]] = own_pages
        slots.append((own_pages.long()[:, None] * page + torch.arange(page, device=DEVICE)).reshape(-1)[:n])
        at += need[i]
    return sum(need) + 2, table, slots


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    kv, q = _lengths(case)
    pages, table, slots = _layout(case, gen)
    s = {"case": case, "pages": pages, "table": table}
    if case["kind"] == "attend":
        s["q"] = _rows(gen, sum(q), case["heads"], case["dim"], dtype)
        s["slots"] = torch.cat(slots).to(torch.int32)
    else:                                            # the new tokens are the last of each sequence
        s["slots"] = torch.cat([v[n - k:] for v, n, k in zip(slots, kv, q)]).to(torch.int32)
    heads = case.get("kv_heads", case["heads"])
    if case.get("fused"):                            # [tokens, queries | keys | values]
        qkv = _rows(gen, sum(q), 4 * heads, case["dim"], dtype)
        s["k"], s["v"] = qkv[:, 2 * heads:3 * heads], qkv[:, 3 * heads:]
    else:
        n = s["slots"].numel()
        s["k"], s["v"] = _rows(gen, n, heads, case["dim"], dtype), _rows(gen, n, heads, case["dim"], dtype)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    kv, q = _lengths(case)
    heads, dim, bits = case.get("kv_heads", case["heads"]), case["dim"], case["bits"]
    if case["kind"] == "attend":
        s["out"] = torch.empty_like(s["q"])
        s["kv_lens"] = torch.tensor(kv, dtype=torch.int32, device=DEVICE)
        starts = [0]
        for n in q:
            starts.append(starts[-1] + n)
        s["q_starts"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE)
    else:
        s["k_out"] = torch.empty(s["k"].shape, dtype=s["k"].dtype, device=DEVICE)
        s["v_out"] = torch.empty_like(s["k_out"])
    if own:
        from tpu_compiler_amd import capi, kv_cache
        global _context
        if _context is None:
            _context = capi.Context(stream=torch.cuda.current_stream().cuda_stream)
        cache = s["cache"] = kv_cache.KVCache(_context, s["pages"], heads, dim, bits=bits, page_tokens=case["page"])
        if case["kind"] == "attend":
            s["attend"] = cache.plan_attention(s["q"], s["out"], s["q_starts"], s["kv_lens"], s["table"], max_q=max(q), max_kv=max(kv),
                                               window=case["window"], sinks=case["sinks"])
        else:
            s["read"] = cache.plan_read(s["slots"], s["k_out"], s["v_out"])
            s["write"] = cache.plan_write(s["k"], s["v"], s["slots"])
        if case["kind"] != "store":
            cache.write(s["k"], s["v"], s["slots"])
    else:
        width = (dim * bits + 7) // 8
        held = s["held"] = [torch.zeros(s["pages"] * case["page"], heads, width, dtype=torch.uint8, device=DEVICE) for _ in range(2)]
        params = s["params"] = [torch.zeros(s["pages"] * case["page"], heads, 2, dtype=torch.bfloat16, device=DEVICE) for _ in range(2)]
        if case["kind"] != "store":
            for a in range(0, s["slots"].numel(), 1 << 16):
                part = slice(a, a + (1 << 16))
                for x, codes, param in zip((s["k"], s["v"]), held, params):
                    codes[s["slots"][part].long()], param[s["slots"][part].long()] = _quantised(x[part], bits)
        if case["kind"] == "attend":
            s["row_seq"] = torch.repeat_interleave(torch.arange(len(q), device=DEVICE), torch.tensor(q, device=DEVICE))
    if case["kind"] != "store":
        del s["k"], s["v"]
    return s


# ---- the plain form --------------------------------------------------------------------------------------------------
def _bf16_down(x):
    """the largest bfloat16 that is not above a float32: the upper half of its bits, of a negative number rounded away from zero"""
    b = x.view(torch.int32)
    return ((b + ((b >> 31) & 0xFFFF)) & -65536).view(torch.float32)


def _quantised(x, bits):
    """the rows' integers, packed, and their offsets and steps"""
    x, top = x.float(), 2 ** bits - 1
    m = _bf16_down(x.amin(-1, keepdim=True))
    s = -_bf16_down(-((x.amax(-1, keepdim=True) - m) / torch.full_like(m, top)))   # by a number, torch multiplies with its inverse
    s = torch.where(s < 2.0 ** -126, 0.0, s)
    c = torch.where(s > 0, ((x - m) / s).round().clamp(0, top), 0.0).to(torch.uint8)
    if bits == 4:
        if c.shape[-1] % 2:
            c = torch.nn.functional.pad(c, (0, 1))
        c = c[..., 0::2] | (c[..., 1::2] << 4)
    return c, torch.cat([m, s], -1).to(torch.bfloat16)


def _read_back(codes, params, bits, dim):
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., :dim]
    p = params.float()
    return p[..., :1] + p[..., 1:] * codes.float()


def _plain_attention(s):
    case = s["case"]
    window, sinks, page, dim, group = case["window"], case["sinks"], case["page"], case["dim"], case["heads"] // case["kv_heads"]
    most_q, most_kv, n = case["q_max"], max(case["kv_max"], case["q_max"]), case["seqs"]
    kv, starts = s["kv_lens"].long(), s["q_starts"].long()
    q_len = starts[1:] - starts[:-1]
    # the positions that any query of a sequence may see: all of them, or the first few and the last ones
    if window and sinks + window + most_q < most_kv:
        first = torch.arange(sinks, device=DEVICE).expand(n, sinks)
        last = kv[:, None] - (window + most_q) + torch.arange(window + most_q, device=DEVICE)
        pos = torch.cat([first, torch.where(last < sinks, -1, last)], 1)
    else:
        pos = torch.arange(most_kv, device=DEVICE).expand(n, most_kv)
    fine = (pos >= 0) & (pos < kv[:, None])
    at = torch.where(fine, pos, 0)
    slots = torch.gather(s["table"].long(), 1, at // page) * page + at % page
    k, v = (_read_back(c[slots], p[slots], case["bits"], dim) for c, p in zip(s["held"], s["params"]))
    i = torch.arange(most_q, device=DEVICE)
    rows = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(n, most_q, case["kv_heads"], group, dim).permute(0, 2, 3, 1, 4).reshape(n, case["kv_heads"], -1, dim)
    scores = torch.matmul(q * dim ** -0.5, k.permute(0, 2, 3, 1).contiguous()).view(n, case["kv_heads"], group, most_q, -1)
    del k
    p = (kv - q_len)[:, None] + i                    # [n, most_q]: where the queries stand
    seen = fine[:, None] & (pos[:, None] <= p[:, :, None])
    if window:
        seen &= (pos[:, None] > p[:, :, None] - window) | (pos[:, None] < sinks)
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.flatten(2, 3), v.permute(0, 2, 1, 3).contiguous()).view(n, case["kv_heads"], group, most_q, dim)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(n, most_q, case["heads"], dim)
    inside = torch.arange(s["q"].shape[0], device=DEVICE) - starts[s["row_seq"]]
    return out[s["row_seq"], inside].to(s["q"].dtype)


def run(s):
    kind = s["case"]["kind"]
    if own:
        if kind == "attend":
            s["attend"]()
            return s["out"]
        if kind == "store":
            s["write"]()
        s["read"]()
        return s["k_out"], s["v_out"]
    if kind == "attend":
        return _plain_attention(s)
    bits, dim, slots = s["case"]["bits"], s["case"]["dim"], s["slots"].long()
    if kind == "store":
        for x, codes, params in zip((s["k"], s["v"]), s["held"], s["params"]):
            codes[slots], params[slots] = _quantised(x, bits)
    return tuple(_read_back(c[slots], p[slots], bits, dim).to(s["k_out"].dtype) for c, p in zip(s["held"], s["params"]))


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def _value64(x, bits):
    """what the cache makes of rows, by the definition: bfloat16 numbers have 8 bits, so m and s are multiples of a power of two"""
    x, top = x.double(), 2 ** bits - 1

    def grid(v):                                     # the distance of bfloat16 numbers around v
        return (v.abs().clamp(min=2.0 ** -126).view(torch.int64) & (0x7FF << 52)).view(torch.float64) / 128

    low = x.min(-1, keepdim=True).values
    m = torch.floor(low / grid(low)) * grid(low)
    step = (x.max(-1, keepdim=True).values - m) / torch.full_like(m, top)
    s = torch.ceil(step / grid(step)) * grid(step)
    c = torch.where(s >= 2.0 ** -126, torch.round((x - m) / s.clamp(min=2.0 ** -126)), 0).clamp(0, top)
    return m + s * c


def exact(case, seed):
    s = _inputs(case, seed)
    bits, kv, q = case["bits"], *_lengths(case)
    if case["kind"] != "attend":
        return _value64(s["k"], bits), _value64(s["v"], bits)
    heads, kv_heads, window, sinks = case["heads"], case["kv_heads"], case["window"], case["sinks"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    row = token = 0
    for n, count in zip(kv, q):
        for a in range(0, count, 512):               # some of a sequence's queries at a time
            b = min(count, a + 512)
            p = torch.arange(n - count + a, n - count + b, device=DEVICE)[:, None]
            t = torch.arange(n, device=DEVICE)
            if window:                               # those that none of them sees are left out
                t = t[(t < sinks) | (t > n - count + a - window)]
            seen = (t <= p) & ((t > p - window) | (t < sinks)) if window else t <= p
            for h in range(kv_heads):
                k, v = _value64(s["k"][token + t, h], bits), _value64(s["v"][token + t, h], bits)
                group = slice(h * heads // kv_heads, (h + 1) * heads // kv_heads)
                x = torch.einsum("qhd,td->qht", s["q"][row + a:row + b, group].double(), k) / case["dim"] ** 0.5
                w = torch.softmax(x.masked_fill(~seen[:, None], float("-inf")), -1)
                out[row + a:row + b, group] = torch.einsum("qht,td->qhd", w, v)
        row, token = row + count, token + n
    return out
