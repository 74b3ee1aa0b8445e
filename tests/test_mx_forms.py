"""Which kernels the products of microscaled numbers launch: tests/cpp/mx_forms.cpp, built by __graft_entry__.build(), stands in for the runtime,
so no device is needed."""
import os
import subprocess

import pytest

import mx_forms

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "mx_forms.bin")


def launches(*lines):
    """each call's kernels and workgroups, as one text"""
    assert os.path.exists(BIN), "build it with __graft_entry__.build()"
    res = subprocess.run([BIN], input="".join(line + "\n" for line in lines), stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=100)
    assert res.returncode == 0, "%d %s" % (res.returncode, res.stderr)
    return res.stdout.splitlines()


# a few rows in one launch, rows that are quantised before, sums in one part
@pytest.mark.parametrize("first", ["product 1 4096 1000 0 0", "linear 1 4096 1000 0 0", "linear 300 4096 5000 1 0", "product 300 512 5000 2 1"])
def test_a_context_has_memory_for_parts_from_its_first_product_on(first):
    """sums that are recorded then are shared by as many workgroups as those of the same call by itself: the same bits"""
    shared = "product 40 16384 1000 0 0"
    alone, = launches(shared)
    assert alone == "mx_tile_kernel<32,64,1,2,4> 128"          # 16 x 2 tiles in four parts
    assert launches("context", first, "capture 1", shared, "capture 0", shared)[3::2] == [alone, alone]


@pytest.mark.parametrize("form,parts,rows,cols,n", mx_forms.CASES)
def test_sizes_take_the_forms_that_they_are_to_test(form, parts, rows, cols, n):
    bm, bn = (int(v) for v in form.split(",")[:2])
    works = parts * -(-rows // bm) * -(-n // bn)
    for dtype in range(3):
        for residual in range(2):
            size = "%d %d %d %d %d" % (rows, cols, n, dtype, residual)
            product, linear = launches("product " + size, "linear " + size)
            assert product == "mx_tile_kernel<%s> %d" % (form, works)
            assert linear.split()[::2] == ["mx_quantize_kernel", "mx_tile_kernel<%s>" % form] and linear.split()[3] == str(works)


def test_every_form_and_number_of_parts_is_tested():
    """what the sizes between one and some hundred thousand rows, numbers and columns take"""
    sizes = [(rows, cols, n) for rows in (17, 40, 70, 200, 600, 2000, 7000, 30000) for cols in (64, 1000, 4000, 20000, 65000, 200000)
             for n in (30, 100, 300, 1000, 4000, 16000, 65536, 300000)]
    sizes += [(39, 190000, 2088), (370, 74000, 998), (51, 92663, 9557)]
    for (rows, _, n), line in zip(sizes, launches(*("product %d %d %d 0 0" % size for size in sizes))):
        kernel, works = line.split()
        form = kernel[len("mx_tile_kernel<"):-1]
        bm, bn = (int(v) for v in form.split(",")[:2])
        parts = int(works) / (-(-rows // bm) * -(-n // bn))
        assert any(form == f and p / 2 < parts <= p for f, p in mx_forms.SIZES), (line, rows, n)


@pytest.mark.parametrize("waves,groups,rows,cols,n", mx_forms.FEW_CASES)
def test_few_rows_take_the_forms_that_they_are_to_test(waves, groups, rows, cols, n):
    for dtype in range(3):
        size = "%d %d %d %d 1" % (rows, cols, n, dtype)
        product, linear = launches("product " + size, "linear " + size)
        for line, of in ((product, -1), (linear, dtype)):
            assert line.split()[::2] == ["mx_stream_kernel<%d,%d,%s>" % (waves, of, str(groups).lower())]
