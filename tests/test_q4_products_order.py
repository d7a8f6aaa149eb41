"""The products around the attention, launched one behind the other: what a kernel may do while the kernel before it still runs,
several host threads at once, and the one order of the sums."""
import os
import re

import numpy as np
import pytest

from tests.test_q4_products import ctx, dev, matrix, packed  # noqa: F401  (ctx, dev: fixtures)

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gwenedeg_b200", "csrc")


def source(name):
    """A source file without its comments."""
    txt = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", txt, flags=re.S))


# ---- a kernel beside the kernel before it -----------------------------------------------------------------------------
def test_rows_are_not_read_as_constants():
    """A product may start while the kernel that writes its rows still runs: levels and scales of rows must not go through the
    read-only path, which no run on a device can be relied on to show."""
    code = source("q4_mm.cuh")
    for call in re.findall(r"(?:__ldg|ldg_stream8?)\(([^;]*);", code):
        assert not re.search(r"\ba\.x[qs]\b", call), call


def test_tensor_memory_is_taken_after_the_wait_and_before_the_next_kernel():
    """Otherwise a kernel that holds tensor memory could wait for one that needs it."""
    code = source("q4_mm.cuh")
    code = code[code.index("q4_tiles_kernel(const"):code.index("cudaError_t launch_q4_tiles")]
    at = [code.index(x) for x in ("pdl_wait()", "tcgen05.alloc", "pdl_launch_dependents()", "setmaxnreg_inc")]
    assert at == sorted(at)
    assert code.count("pdl_wait()") == code.count("tcgen05.alloc") == code.count("pdl_launch_dependents()") == 1


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 40, 100, 300])
def test_norm_and_product_in_turn_on_the_same_rows_without_a_wait(ctx, dev, rows):
    """The same 8-bit rows are written and read again and again with other values, nothing waiting in between: the bits of calls that
    are waited for one by one."""
    rng = np.random.default_rng(rows)
    k, n, gs, eps, turns = 1088, 264, 32, 1e-6, 12
    w = ctx.q4_new(*(lambda m: (packed(m[0]), m[1]))(matrix(rng, n, k, gs)), gs)
    xs = [dev.put((rng.standard_normal((rows, k)) * 4.0 ** (i % 5)).astype(np.float32)) for i in range(turns)]
    pw = dev.put(np.ones(k, np.float32) * np.float32(0.7))
    q, s = dev.room((rows, k), np.int8), dev.room((rows, k // gs), np.float32)
    outs = [dev.room((rows, n), np.float32) for _ in range(turns)]
    alone = []
    for i in range(turns):
        ctx.add_norm_quant_dev(rows, k, gs, xs[i], None, pw, eps, None, None, q, s)
        ctx.sync()
        ctx.mm_q4_dev(w, rows, q, s, outs[i])
        alone.append(dev.get(outs[i], (rows, n)))
    assert all(not np.array_equal(alone[0], a) for a in alone[1:])
    for _ in range(20):
        for i in range(turns):
            ctx.add_norm_quant_dev(rows, k, gs, xs[i], None, pw, eps, None, None, q, s)
            ctx.mm_q4_dev(w, rows, q, s, outs[i])
    for i in range(turns):
        assert np.array_equal(dev.get(outs[i], (rows, n)).view(np.uint32), alone[i].view(np.uint32)), i
