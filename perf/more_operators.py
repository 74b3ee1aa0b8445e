"""The language-model operators around the key/value cache that performance is measured on: weights and activations as microscaled
4-bit floating point numbers, their products, and the pages that a batch's sequences have in a cache.

  quantise  rows become 4-bit numbers with a scale for each 32 of them, and are read back
  product   y = x w^T (+ bias) (+ residual) with w in 4 bits; x rows of 16 or 32 bits that the call quantises, or in 4 bits already
  pages     tokens that a batch no longer has are taken off its page table, new ones get pages and slots

A row is held in blocks of 32 numbers, the last one filled up with zeros.  A block has a scale 2^e, e = floor(log2(its largest size)) - 2
in -127..127 (-127 for zeros), a byte e + 127, and codes of 4 bits, sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6: the nearest to
x / 2^e, a tie to the code that is even, the largest for what is beyond.  Even columns are the low halves of their bytes.

`own` chooses between the framework's operators and their plain form in torch, in 32 bits."""
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEVICE = "cuda"
BLOCK = 32
_context = None


# ---- cases -----------------------------------------------------------------------------------------------------------
def _quantise(name, rows, cols, dtype, part=False):
    """part: the rows are a part of longer ones"""
    return dict(name=name, kind="quantise", rows=rows, cols=cols, dtype=dtype, part=part)


def _product(name, rows, k, cols, dtype, ready=False, bias=False, residual=False):
    """ready: x is in 4 bits before the call"""
    return dict(name=name, kind="product", rows=rows, k=k, cols=cols, dtype=dtype, ready=ready, bias=bias, residual=residual)


def _pages(name, seqs, held, new, page, short=False):
    """`seqs` sequences of 0..held tokens that get 0..new tokens (new = 1: each one); short: fewer pages than they need"""
    return dict(name=name, kind="pages", seqs=seqs, held=held, new=new, page=page, short=short)


def listed():
    return [
        # a token's activations on their way to another program (latency)
        _quantise("quant_token", 1, 4096, "bf16"),
        # a long prompt's activations
        _quantise("quant_prompt", 8192, 8192, "bf16"),
        # a layer's weights as training left them: float32, an odd width, rows that are parts of longer ones
        _quantise("quant_weights", 4999, 2050, "f32", part=True),
        # one user's next token through a layer (latency), and through the layer that gives its logits
        _product("token", 1, 4096, 4096, "bf16", residual=True),
        _product("token_logits", 1, 4096, 65536, "f32"),
        # a few tokens at once (a draft to be checked), the sizes of a classifier, float16
        _product("draft", 6, 2048, 1000, "f16", bias=True),
        # a batch's next tokens, up (activations in 4 bits, shared by several products) and down a wide layer
        _product("batch_up", 64, 4096, 16384, "bf16", ready=True),
        _product("batch_down", 48, 16384, 4096, "bf16", residual=True),
        # part of a prompt, odd sizes everywhere
        _product("chunk", 777, 2050, 4999, "f32", bias=True, residual=True),
        # a prompt
        _product("prompt", 8192, 8192, 8192, "bf16"),
        # every step of generation: a token for each sequence of a batch (latency)
        _pages("pages_step", 64, 8000, 1, 64),
        # requests come and go: prompts for a large batch
        _pages("pages_prompts", 700, 3000, 900, 32),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("quantise", "product", "product", "product", "pages"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "quantise":
        cols = rng.choice((_log(rng, 1, 20000), BLOCK * _log(rng, 1, 500)))
        case = _quantise("", _log(rng, 1, 8192), cols, dtype, part=rng.random() < 0.4)
    elif kind == "product":
        form = rng.choice(("token", "few", "batch", "prompt"))
        rows = 1 if form == "token" else _log(rng, 2, 16) if form == "few" else _log(rng, 17, 256) if form == "batch" else _log(rng, 257, 8192)
        k = rng.choice((_log(rng, 32, 16384), BLOCK * _log(rng, 4, 512)))
        cols = rng.choice((_log(rng, 16, 65536), 64 * _log(rng, 1, 512)))
        case = _product("", rows, k, cols, dtype, ready=rng.random() < 0.25, bias=rng.random() < 0.4, residual=rng.random() < 0.4)
    else:
        case = _pages("", _log(rng, 1, 1000), rng.choice((0, _log(rng, 10, 10000))), rng.choice((1, _log(rng, 1, 1000))),
                      rng.choice((32, 64, 128, 96)), short=rng.random() < 0.2)
    del case["name"]
    top = {"quantise": "quant_prompt", "product": "prompt", "pages": "pages_prompts"}[kind]
    limit = _cost(next(c for c in listed() if c["name"] == top))
    while _cost(case) > limit:                       # no more than the largest listed one
        most = max((k for k in ("rows", "cols", "k", "seqs", "held", "new") if k in case), key=case.get)
        case[most] = (case[most] + 1) // 2
    return case


def _cost(case):
    """what draw() bounds: bytes, or of products the operations, a byte counted as 1900 of them"""
    w = work(case)
    return max(w["flops"], 1900 * w["bytes"]) if case["kind"] == "product" else w["bytes"]


def _sequences(case):
    """tokens that each sequence holds, tokens that it gets"""
    rng = random.Random(case["seqs"] * 7 + case["held"])
    held = [rng.choice((0, rng.randint(0, case["held"]), rng.randint(0, case["held"]))) for _ in range(case["seqs"])]
    new = [1 if case["new"] == 1 else rng.choice((0, 1, rng.randint(0, case["new"]), case["new"])) for _ in range(case["seqs"])]
    return held, new


def _pool(case):
    """pages of the cache, pages that a row of the table has room for, slots that a step has room for"""
    held, new = _sequences(case)
    page = case["page"]
    before = sum(-(-h // page) for h in held)
    after = sum(-(-(h + n) // page) for h, n in zip(held, new))
    pages = before + (after - before) // 2 if case["short"] else after + 3
    return max(1, pages), max(1, max(-(-(h + n) // page) for h, n in zip(held, new))), max(1, sum(new))


def _held(rows, cols):
    return rows * -(-cols // BLOCK) * 17             # 16 bytes of codes and one of scale a block


def work(case):
    if case["kind"] == "pages":
        held, new = _sequences(case)
        page = case["page"]
        taken = sum(-(-(h + n) // page) - -(-h // page) for h, n in zip(held, new))
        # both calls: lengths and wishes read, lengths written, a table entry and a place of the free pages for each page; starts; slots
        return {"bytes": 4 * (2 * 3 * len(held) + 2 * 2 * taken + len(held) + 1 + sum(new)), "flops": 0}
    size = TYPES[case["dtype"]].itemsize
    if case["kind"] == "quantise":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * size + 2 * _held(case["rows"], case["cols"]), "flops": 12 * n}
    rows, k, cols = case["rows"], case["k"], case["cols"]
    x = _held(rows, k) if case["ready"] else rows * k * size
    return {"bytes": x + _held(cols, k) + rows * cols * size * (2 if case["residual"] else 1) + (4 * cols if case["bias"] else 0),
            "flops": 2 * rows * k * cols}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _activations(gen, rows, cols, dtype):
    """as layers produce them: channels of different size, a few of them far larger than the rest"""
    size = torch.rand(cols, generator=gen, device=DEVICE) * 1.5 + 0.25
    size *= torch.where(torch.rand(cols, generator=gen, device=DEVICE) < 0.01, 20.0, 1.0)
    x = torch.empty(rows, cols, dtype=dtype, device=DEVICE)
    for a in range(0, rows, 2048):
        b = min(rows, a + 2048)
        x[a:b] = torch.randn(b - a, cols, generator=gen, device=DEVICE) * size
    return x


def _weights(gen, rows, cols):
    """a layer's, rows of different size"""
    size = (torch.rand(rows, 1, generator=gen, device=DEVICE) + 0.5) * cols ** -0.5
    x = torch.randn(rows, cols, generator=gen, device=DEVICE)
    return x.mul_(size)


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "pages":
        pages, _, _ = _pool(case)
        held, new = _sequences(case)
        # pages that are free, in the order of a cache that has been in use for a while; the batch is in another order each time
        s["free"] = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
        order = torch.randperm(len(held), generator=gen, device=DEVICE)
        s["held"], s["new"] = (torch.tensor(v, dtype=torch.int32, device=DEVICE)[order] for v in (held, new))
        return s
    dtype = TYPES[case["dtype"]]
    if case["kind"] == "quantise":
        extra = 31 if case["part"] else 0
        make = _weights if case["dtype"] == "f32" else lambda g, r, c: _activations(g, r, c, dtype)
        s["x"] = make(gen, case["rows"], case["cols"] + extra)[:, extra:]
        return s
    s["x"] = _activations(gen, case["rows"], case["k"], dtype)
    s["w"] = _weights(gen, case["cols"], case["k"])
    if case["bias"]:
        s["bias"] = torch.randn(case["cols"], generator=gen, device=DEVICE)
    if case["residual"]:
        s["residual"] = _activations(gen, case["rows"], case["cols"], dtype)
    return s


def _own_context():
    from tpu_compiler_amd import capi
    global _context
    if _context is None:
        _context = capi.Context(stream=torch.cuda.current_stream().cuda_stream)
    return _context


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "pages":
        return _prepare_pages(s)
    if case["kind"] == "quantise":
        s["out"] = torch.empty(case["rows"], case["cols"], dtype=s["x"].dtype, device=DEVICE)
        shape = case["rows"], case["cols"]
        s["codes"] = torch.zeros(shape[0], -(-shape[1] // BLOCK) * 16, dtype=torch.uint8, device=DEVICE)
        s["scales"] = torch.zeros(shape[0], -(-shape[1] // BLOCK), dtype=torch.uint8, device=DEVICE)
        if own:
            from tpu_compiler_amd import mx
            m = mx.MXMatrix(_own_context(), *shape, codes=s["codes"], scales=s["scales"])
            s["quantize"], s["read"] = m.plan_quantize(s["x"]), m.plan_read(s["out"])
        return s
    s["out"] = torch.empty(case["rows"], case["cols"], dtype=s["x"].dtype, device=DEVICE)
    s["w"] = _quantised(s["w"])                      # as a file of weights holds them
    if case["ready"]:
        s["x"] = _quantised(s["x"])
    if own:
        from tpu_compiler_amd import mx
        ctx = _own_context()
        w = mx.MXMatrix(ctx, case["cols"], case["k"], codes=s["w"][0], scales=s["w"][1])
        x = mx.MXMatrix(ctx, case["rows"], case["k"], codes=s["x"][0], scales=s["x"][1]) if case["ready"] else s["x"]
        s["product"] = mx.plan_product(ctx, x, w, s["out"], bias=s.get("bias"), residual=s.get("residual"))
    return s


def _prepare_pages(s):
    """the batch as a pass begins: it has the tokens that go and come"""
    case = s["case"]
    pages, most, room = _pool(case)
    n = case["seqs"]
    s["lens"] = torch.zeros(n, dtype=torch.int32, device=DEVICE)
    s["table"] = torch.full((n, most), -1, dtype=torch.int32, device=DEVICE)
    s["n_free"] = torch.full((1,), pages, dtype=torch.int32, device=DEVICE)
    s["q_starts"] = torch.zeros(n + 1, dtype=torch.int32, device=DEVICE)
    s["slots"] = torch.zeros(max(room, sum(_sequences(case)[0])), dtype=torch.int32, device=DEVICE)
    s["refused"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    _grow(s, s["held"])
    s["slots"] = torch.zeros(room, dtype=torch.int32, device=DEVICE)
    _grow(s, s["new"])
    if own:
        from tpu_compiler_amd import kv_cache
        p = kv_cache.KVPages(_own_context(), pages, n, most, page_tokens=case["page"], lens=s["lens"], table=s["table"], free=s["free"],
                             n_free=s["n_free"])
        s["trim"] = p.plan_trim(s["held"])
        s["grow"] = p.plan_grow(s["new"], s["q_starts"], s["slots"], s["refused"])
    return s


# ---- the plain form --------------------------------------------------------------------------------------------------
def _power(e):
    """2^(e - 127), e in 0..254"""
    return torch.where(e > 0, e << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _quantised(x):
    """rows as codes, two in a byte, and scales"""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    top = x.abs().amax(-1, keepdim=True)
    e = (top.view(torch.int32) >> 23).clamp(min=2) - 2                  # the exponent's bits: of zeros and the smallest numbers 0
    size = x.abs() * _power(254 - e)
    # the middles between codes; a middle belongs to the even one of the two
    code = sum((size > b if i % 2 == 0 else size >= b).to(torch.uint8) for i, b in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)))
    code |= torch.signbit(x).to(torch.uint8) << 3
    code = code.view(rows, -1)
    return code[:, 0::2] | code[:, 1::2] << 4, e.view(rows, -1).to(torch.uint8)


def _values(codes, scales, cols):
    """what they stand for, in 32 bits"""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=DEVICE)
    x = table[torch.stack([codes & 15, codes >> 4], -1).int()].view(codes.shape[0], -1, BLOCK)
    return (x * _power(scales.int())[..., None]).view(codes.shape[0], -1)[:, :cols]


def _grow(s, new):
    """new tokens for sequences in order.  One gets its tokens if the table's row has room for them, the step has for all wishes up to its own, and the
    pages that it needs are there after those that the ones before it need."""
    page, (n, most) = s["case"]["page"], s["table"].shape
    lens, new, free, n_free = s["lens"].long(), new.long(), s["free"], s["n_free"].long()
    fits = lens + new <= most * page
    have = (lens + page - 1) // page
    need = torch.where(fits, (lens + new + page - 1) // page - have, 0)
    upto = torch.cumsum(need, 0)
    served = fits & (torch.cumsum(torch.where(fits, new, 0), 0) <= s["slots"].numel()) & ((need == 0) | (upto <= n_free))
    add, take = torch.where(served, new, 0), torch.where(served, need, 0)
    ends = torch.cumsum(add, 0)
    s["q_starts"][1:] = ends
    s["refused"][:] = ((new > 0) & ~served).sum()
    col = torch.arange(most, device=DEVICE) - have[:, None]             # of the new pages
    at = n_free - 1 - (upto - need)[:, None] - col
    s["table"].copy_(torch.where((col >= 0) & (col < take[:, None]), free[at.clamp(0, free.numel() - 1)], s["table"]))
    t = torch.arange(s["slots"].numel(), device=DEVICE)
    seq = torch.searchsorted(ends, t, right=True).clamp(max=n - 1)
    pos = (lens - ends + add)[seq] + t
    slot = s["table"][seq, (pos // page).clamp(0, most - 1)].long() * page + pos % page
    s["slots"].copy_(torch.where(t < ends[-1], slot, -1))
    s["lens"] += add.to(torch.int32)
    s["n_free"] -= take.sum().to(torch.int32)


def _trim(s, keep):
    """the sequences' tokens from `keep` on go; the next to grow gets the pages as these got them"""
    page, most, n_free, lens = s["case"]["page"], s["table"].shape[1], s["n_free"].long(), s["lens"].long()
    keep = torch.minimum(keep.long(), lens)
    have, left = (lens + page - 1) // page, (keep + page - 1) // page
    upto = torch.cumsum(have - left, 0)
    col = torch.arange(most, device=DEVICE) - left[:, None]
    gone = (col >= 0) & (col < (have - left)[:, None])
    at = n_free + upto[-1] - 1 - (upto - have + left)[:, None] - col
    free = torch.cat([s["free"], s["free"].new_zeros(1)])               # a place for what stays
    free.scatter_(0, torch.where(gone, at, free.numel() - 1).view(-1), s["table"].view(-1))
    s["free"].copy_(free[:-1])
    s["table"].masked_fill_(gone, -1)
    s["n_free"] += upto[-1].to(torch.int32)
    s["lens"].copy_(keep)


def run(s):
    case = s["case"]
    if case["kind"] == "pages":
        if own:
            s["trim"]()
            s["grow"]()
        else:
            _trim(s, s["held"])
            _grow(s, s["new"])
        return {k: s[k] for k in ("lens", "table", "free", "n_free", "q_starts", "slots", "refused")}
    if case["kind"] == "quantise":
        if own:
            s["quantize"]()
            s["read"]()
            return s["out"]
        return _values(*_quantised(s["x"]), case["cols"]).to(s["out"].dtype)
    if own:
        s["product"]()
        return s["out"]
    x = s["x"] if case["ready"] else _quantised(s["x"])
    y = _values(*x, case["k"]) @ _values(*s["w"], case["k"]).t()
    if case["bias"]:
        y += s["bias"]
    if case["residual"]:
        y += s["residual"].float()
    return y.to(s["out"].dtype)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def _value64(x):
    """what rows stand for in 4 bits, by the definition: between 2^a and 2^(a + 1) numbers of one fraction bit lie 2^(a - 1) apart, and those
    below 1 lie 1/2 apart"""
    rows, cols = x.shape
    out = torch.empty(rows, cols, dtype=torch.float64, device=x.device)
    for a in range(0, cols, BLOCK * 64):
        part = x[:, a:a + BLOCK * 64].double()
        width = part.shape[1]
        part = torch.cat([part, part.new_zeros(rows, -width % BLOCK)], 1).unflatten(1, (-1, BLOCK))
        e = (torch.frexp(part.abs().max(-1, keepdim=True).values)[1] - 1 - 2).clamp(-127, 127)    # frexp's fraction is below 1
        scale = (e.long() + 1023 << 52).view(torch.float64)
        v = part / scale
        grid = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
        out[:, a:a + width] = ((torch.round(v / grid) * grid).clamp(-6, 6) * scale).flatten(1)[:, :width]
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "pages":
        return None                                  # whole numbers
    if case["kind"] == "quantise":
        return _value64(s["x"])
    x, w = _value64(s["x"]), _value64(s["w"])
    y = torch.empty(case["rows"], case["cols"], dtype=torch.float64, device=DEVICE)
    for a in range(0, case["cols"], 4096):
        y[:, a:a + 4096] = torch.matmul(x, w[a:a + 4096].t())
    if case["bias"]:
        y += s["bias"].double()
    if case["residual"]:
        y += s["residual"].double()
    return y
