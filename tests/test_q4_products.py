"""The products around the attention: residual + RMS norm + 8-bit rows, 8-bit rows times 4-bit matrices, the gated feed-forward
product.  Against the definitions in 64 bits, with bounds derived from the operations: every fp32 operation is off by at
most half a step (2^-24 relative), and a sum's error is bounded by its number of operations times the sum of the magnitudes."""
import ctypes as C

import numpy as np
import pytest

U = 2.0 ** -24  # half a step of fp32, relative
SLICE = 512


def matrix(rng, n, k, gs):
    lev = rng.integers(-8, 8, (n, k)).astype(np.int8)
    sc = (rng.uniform(0.2, 1.0, (n, k // gs)) * 0.01).astype(np.float16)
    return lev, sc


def packed(lev):
    u = (lev + 8).astype(np.uint8)
    return np.ascontiguousarray(u[:, 0::2] | (u[:, 1::2] << 4))


def rows8(rng, rows, k, gs):
    xq = rng.integers(-127, 128, (rows, k)).astype(np.int8)
    xs = rng.uniform(0.001, 0.05, (rows, k // gs)).astype(np.float32)
    return xq, xs


def product(xq, xs, lev, sc, gs):
    """(y, bound on the fp32 result's error): sum_g xs ws D with D exact.  The scale product is rounded once, a term passes through
    at most 512 / gs multiply-adds and as many additions as there are slices, each half a step of something no larger than
    the sum of the terms' magnitudes; 1.01 covers the products of these factors."""
    r, k = xq.shape
    n, G = lev.shape[0], k // gs
    D = np.einsum("rgi,ngi->rng", xq.reshape(r, G, gs).astype(np.float64), lev.reshape(n, G, gs).astype(np.float64), optimize=True)
    t = D * xs.astype(np.float64)[:, None, :] * sc.astype(np.float64)[None]
    ops = 1 + min(G, SLICE // gs) + -(-k // SLICE)
    return t.sum(2), 1.01 * ops * U * np.abs(t).sum(2)


def quantised(x, gs):
    """The library's quantiser on fp32 rows, operation for operation in fp32."""
    g = np.ascontiguousarray(x, np.float32).reshape(x.shape[0], -1, gs)
    top = np.abs(g).max(2, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(top > 0, np.float32(127.0) / top, np.float32(0))
        v = g * inv
    lev = np.trunc(v + np.copysign(np.float32(0.49999997), v)).astype(np.int8)
    return lev.reshape(x.shape), top[..., 0]


@pytest.fixture
def ctx():
    import gwenedeg_b200 as g
    c = g.Context(0, n_attn=1, n_heads=8, n_kv_heads=2, head_dim=128, max_rows=512)
    yield c
    c.close()


class Dev:
    """Device buffers of one test."""

    def __init__(self, c):
        self.c, self.held = c, []

    def put(self, a):
        self.held.append(self.c.to_device(a))
        return self.held[-1]

    def room(self, shape, dtype, fill=None):
        a = np.zeros(shape, dtype) if fill is None else np.full(shape, fill, dtype)
        return self.put(a)

    def get(self, p, shape, dtype=np.float32):
        a = np.empty(shape, dtype)
        self.c.d2h(a, p)
        self.c.sync()
        return a

    def free(self):
        for p in self.held:
            self.c.mfree(p)


@pytest.fixture
def dev(ctx):
    d = Dev(ctx)
    yield d
    d.free()


# ---- without a GPU ----------------------------------------------------------------------------------------------------
def test_entry_points_refuse_a_missing_context():
    import gwenedeg_b200 as g
    L = g._lib.load()
    buf, out = (C.c_ubyte * 256)(), C.c_void_p()
    b = C.cast(buf, C.c_void_p)
    assert L.rq_cuda_q4_new(None, 1, 32, 32, b, b, C.byref(out)) == -1
    assert L.rq_cuda_q4_new_dev(None, 1, 32, 32, b, b, C.byref(out)) == -1
    assert L.rq_cuda_add_norm_quant_dev(None, 1, 32, 32, b, None, b, 1e-6, None, b, None, None) == -1
    assert L.rq_cuda_mm_q4_dev(None, None, 1, b, b, b) == -1
    assert L.rq_cuda_ffn_q4_dev(None, None, None, 1, b, b, b, None, None) == -1
    assert L.rq_cuda_q4_bytes(None) == 0
    L.rq_cuda_q4_free(None)


def test_the_bound_holds_for_a_product_in_single_precision():
    """The test's own arithmetic: the order the header states, in numpy fp32 with separate multiplications and additions (one more
    rounding per term than fused), stays inside twice the bound."""
    rng = np.random.default_rng(0)
    gs, k = 32, 1120
    lev, sc = matrix(rng, 7, k, gs)
    xq, xs = rows8(rng, 3, k, gs)
    want, tol = product(xq, xs, lev, sc, gs)
    G = k // gs
    D = np.einsum("rgi,ngi->rng", xq.reshape(3, G, gs).astype(np.int64), lev.reshape(7, G, gs).astype(np.int64)).astype(np.float32)
    y = np.zeros((3, 7), np.float32)
    for s in range(0, G, SLICE // gs):
        p = np.zeros((3, 7), np.float32)
        for g in range(s, min(G, s + SLICE // gs)):
            p = p + D[:, :, g] * (sc[None, :, g].astype(np.float32) * xs[:, None, g])
        y = y + p
    assert (np.abs(y - want) <= 2 * tol).all()


# ---- the product ------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,gs", [
    (1, 1, 32, 32), (1, 16, 32, 32), (2, 17, 96, 32), (1, 100, 128, 128), (8, 33, 192, 64), (9, 64, 544, 32), (16, 47, 640, 128),
    (17, 130, 1024, 64), (32, 15, 2080, 32), (33, 129, 4160, 64), (64, 40, 12288, 128), (65, 80, 1056, 32), (130, 257, 2176, 128), (300, 200, 1088, 64),
    (512, 384, 512, 32)])
def test_product_matches_the_definition(ctx, dev, rows, n, k, gs):
    rng = np.random.default_rng(rows * 7 + n + k + gs)
    lev, sc = matrix(rng, n, k, gs)
    xq, xs = rows8(rng, rows, k, gs)
    w = ctx.q4_new(packed(lev), sc, gs)
    guard = 64
    out = dev.room(rows * n + guard, np.float32, fill=-7.5)
    ctx.mm_q4_dev(w, rows, dev.put(xq), dev.put(xs), out)
    got = dev.get(out, rows * n + guard)
    assert (got[rows * n:] == -7.5).all()  # nothing behind the last row
    got = got[:rows * n].reshape(rows, n)
    want, tol = product(xq, xs, lev, sc, gs)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,gs", [(150, 1120, 32), (264, 4224, 128), (144, 1600, 64)])
def test_a_rows_result_does_not_depend_on_the_other_rows(ctx, dev, n, k, gs):
    rng = np.random.default_rng(k)
    most = 300
    lev, sc = matrix(rng, n, k, gs)
    xq, xs = rows8(rng, most, k, gs)
    w = ctx.q4_new(packed(lev), sc, gs)
    q, s = dev.put(xq), dev.put(xs)
    out = dev.room((most, n), np.float32)
    alone = np.empty((most, n), np.float32)
    for r in list(range(0, 70)) + [127, 128, 255, 256, most - 1]:
        ctx.mm_q4_dev(w, 1, q + r * k, s + r * (k // gs) * 4, out)  # (rows start where they start: 32-byte steps)
        alone[r] = dev.get(out, n)
    for rows in (2, 7, 8, 9, 16, 17, 32, 33, 48, 63, 64, 65, 96, 128, 129, 192, 256, 257, most):
        ctx.mm_q4_dev(w, rows, q, s, out)
        got = dev.get(out, (rows, n))
        for r in [x for x in list(range(0, 70)) + [127, 128, 255, 256, most - 1] if x < rows]:
            assert np.array_equal(got[r].view(np.uint32), alone[r].view(np.uint32)), (rows, r)


@pytest.mark.gpu
@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 40, 200])
def test_largest_levels_are_exact(ctx, dev, rows, gs):
    """All levels at their limits: D = gs x 127 x 8, or gs x 128 x 8 for the level -128 that no quantiser here makes."""
    n, k = 32, 512
    for level, xl in ((-8, 127), (-8, -127), (7, 127), (-8, -128)):
        w = ctx.q4_new(packed(np.full((n, k), level, np.int8)), np.full((n, k // gs), 0.5, np.float16), gs)
        out = dev.room((rows, n), np.float32)
        ctx.mm_q4_dev(w, rows, dev.put(np.full((rows, k), xl, np.int8)), dev.put(np.full((rows, k // gs), 2.0, np.float32)), out)
        assert (dev.get(out, (rows, n)) == float(k * level * xl)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 70])
def test_values_that_are_not_finite_stay_in_their_row_and_output(ctx, dev, rows):
    rng = np.random.default_rng(5)
    n, k, gs = 40, 1056, 32
    lev, sc = matrix(rng, n, k, gs)
    xq, xs = rows8(rng, rows, k, gs)
    clean, tol = product(xq, xs, lev, sc, gs)
    sc[5, 3] = np.nan
    sc[20, 32] = np.inf  # (the last group, in a chunk that is not full)
    xs[1, 2] = np.nan
    xs[2, 32] = np.inf
    w = ctx.q4_new(packed(lev), sc, gs)
    out = dev.room((rows, n), np.float32)
    ctx.mm_q4_dev(w, rows, dev.put(xq), dev.put(xs), out)
    got = dev.get(out, (rows, n))
    bad = np.zeros((rows, n), bool)
    bad[[1, 2]] = True
    bad[:, [5, 20]] = True
    assert not np.isfinite(got[bad]).any()
    assert (np.abs(got - clean) <= tol)[~bad].all()


@pytest.mark.gpu
def test_matrix_from_host_and_from_device_memory(ctx, dev):
    rng = np.random.default_rng(6)
    n, k, gs = 37, 320, 64
    lev, sc = matrix(rng, n, k, gs)
    xq, xs = rows8(rng, 5, k, gs)
    a = ctx.q4_new(packed(lev), sc, gs)
    b = ctx.q4_new_dev(n, k, gs, dev.put(packed(lev)), dev.put(sc))
    assert a.nbytes == b.nbytes >= n * k // 2 + sc.nbytes
    q, s = dev.put(xq), dev.put(xs)
    o1, o2 = dev.room((5, n), np.float32), dev.room((5, n), np.float32)
    ctx.mm_q4_dev(a, 5, q, s, o1)
    ctx.mm_q4_dev(b, 5, q, s, o2)
    assert np.array_equal(dev.get(o1, (5, n)), dev.get(o2, (5, n)))
    a.free()
    a.free()  # (nothing left to free)


# ---- the gated product ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,gs", [
    (1, 32, 32, 32), (1, 384, 4096, 64), (5, 17, 96, 32), (8, 256, 1152, 128), (13, 160, 1056, 32), (19, 192, 640, 64), (33, 128, 2176, 128),
    (64, 96, 544, 32), (70, 320, 1600, 64), (129, 384, 512, 128), (260, 64, 1088, 64)])
def test_gated_product_matches_the_definition(ctx, dev, rows, n, k, gs):
    rng = np.random.default_rng(rows + n + k)
    gl, gsc = matrix(rng, n, k, gs)
    ul, usc = matrix(rng, n, k, gs)
    xq, xs = rows8(rng, rows, k, gs)
    xs[:] *= np.float32(0.3)
    g, gt = product(xq, xs, gl, gsc, gs)
    u, ut = product(xq, xs, ul, usc, gs)
    sig = 1.0 / (1.0 + np.exp(-g))
    want = g * sig * u
    # silu'(g) is at most 1.1 in magnitude; e^-g (2 units in the last place = 4 U), 1 + e^-g, the division and the product: at most 7 U
    # of |h|; the second-order term gt * ut is kept
    tol = 1.1 * gt * (np.abs(u) + ut) + (np.abs(g * sig)) * ut + 8 * U * np.abs(want) + 1e-37
    gate, up = ctx.q4_new(packed(gl), gsc, gs), ctx.q4_new(packed(ul), usc, gs)
    q, s = dev.put(xq), dev.put(xs)
    h = dev.room(rows * n + 64, np.float32, fill=-7.5)
    ctx.ffn_q4_dev(gate, up, rows, q, s, h, None, None)
    first = dev.get(h, rows * n + 64)
    assert (first[rows * n:] == -7.5).all()
    first = first[:rows * n].reshape(rows, n)
    assert (np.abs(first - want) <= tol).all(), float((np.abs(first - want) / tol).max())
    if n % gs:
        import gwenedeg_b200 as gw
        with pytest.raises(gw.RqCudaError):
            ctx.ffn_q4_dev(gate, up, rows, q, s, h, h, s)
        return
    # the 8-bit rows are the quantiser's on exactly these fp32 rows, with and without the fp32 rows beside them
    for with_h in (True, False):
        hq = dev.room(rows * n + 64, np.int8, fill=99)
        hs = dev.room(rows * (n // gs) + 64, np.float32, fill=-7.5)
        ctx.ffn_q4_dev(gate, up, rows, q, s, h if with_h else None, hq, hs)
        lev, top = quantised(first, gs)
        gq, gsx = dev.get(hq, rows * n + 64, np.int8), dev.get(hs, rows * (n // gs) + 64)
        assert (gq[rows * n:] == 99).all() and (gsx[rows * (n // gs):] == -7.5).all()
        assert np.array_equal(gq[:rows * n].reshape(rows, n), lev)
        assert np.array_equal(gsx[:rows * (n // gs)].reshape(rows, -1), top * np.float32(1.0 / 127.0))
        if with_h:
            assert np.array_equal(dev.get(h, (rows, n)).view(np.uint32), first.view(np.uint32))


@pytest.mark.gpu
def test_gated_rows_do_not_depend_on_the_other_rows(ctx, dev):
    rng = np.random.default_rng(3)
    n, k, gs, most = 192, 1600, 64, 200
    gl, gsc = matrix(rng, n, k, gs)
    ul, usc = matrix(rng, n, k, gs)
    xq, xs = rows8(rng, most, k, gs)
    gate, up = ctx.q4_new(packed(gl), gsc, gs), ctx.q4_new(packed(ul), usc, gs)
    q, s = dev.put(xq), dev.put(xs)
    h, hq, hs = dev.room((most, n), np.float32), dev.room((most, n), np.int8), dev.room((most, n // gs), np.float32)
    ctx.ffn_q4_dev(gate, up, most, q, s, h, hq, hs)
    all_h, all_q, all_s = dev.get(h, (most, n)), dev.get(hq, (most, n), np.int8), dev.get(hs, (most, n // gs))
    for r0, rows in ((0, 1), (7, 1), (199, 1), (3, 8), (64, 16), (10, 33), (100, 64), (1, 65), (50, 130)):
        ctx.ffn_q4_dev(gate, up, rows, q + r0 * k, s + r0 * (k // gs) * 4, h, hq, hs)
        assert np.array_equal(dev.get(h, (rows, n)).view(np.uint32), all_h[r0:r0 + rows].view(np.uint32)), (r0, rows)
        assert np.array_equal(dev.get(hq, (rows, n), np.int8), all_q[r0:r0 + rows])
        assert np.array_equal(dev.get(hs, (rows, n // gs)), all_s[r0:r0 + rows])


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,gs", [(256, 4224, 128), (160, 2080, 32), (192, 8256, 64)])
def test_gated_rows_in_8_bits_over_every_kernel(ctx, dev, n, k, gs):
    """Few rows, many rows, inputs split over a cluster or not, groups inside a tile and across two: the same bits for the same row; a row
    whose scale is no number stays alone."""
    rng = np.random.default_rng(k + gs)
    most = 300
    gl, gsc = matrix(rng, n, k, gs)
    ul, usc = matrix(rng, n, k, gs)
    xq, xs = rows8(rng, most, k, gs)
    xs *= np.float32(0.3)
    xs[2, 1] = np.nan
    gate, up = ctx.q4_new(packed(gl), gsc, gs), ctx.q4_new(packed(ul), usc, gs)
    q, s = dev.put(xq), dev.put(xs)
    h, hq, hs = dev.room((most, n), np.float32), dev.room((most, n), np.int8), dev.room((most, n // gs), np.float32)
    first = None
    for rows in (1, 3, 8, 9, 24, 56, 57, 64, 65, 100, 128, 129, 200, most):
        ctx.ffn_q4_dev(gate, up, rows, q, s, h, hq, hs)
        got = dev.get(h, (rows, n)), dev.get(hq, (rows, n), np.int8), dev.get(hs, (rows, n // gs))
        if rows == 3:
            first = got
            ok = [0, 1]
            lev, top = quantised(got[0][ok], gs)
            assert np.array_equal(got[1][ok], lev) and np.array_equal(got[2][ok], top * np.float32(1.0 / 127.0))
            assert np.isnan(got[0][2]).all() and (got[1][2] == 0).all() and (got[2][2] == 0).all()
        elif rows > 3:
            for a, b in zip(got, first):
                assert np.array_equal(a[:3].view(np.uint8), b.view(np.uint8)), rows


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,gs", [(1, 48, 20480, 64), (20, 48, 20480, 128), (70, 144, 20480, 32), (130, 144, 12320, 32), (57, 528, 3584, 64), (260, 1040, 1536, 128)])
def test_long_inputs_and_ragged_tiles(ctx, dev, rows, n, k, gs):
    rng = np.random.default_rng(rows + k)
    lev, sc = matrix(rng, n, k, gs)
    xq, xs = rows8(rng, rows, k, gs)
    w = ctx.q4_new(packed(lev), sc, gs)
    out = dev.room((rows, n), np.float32)
    ctx.mm_q4_dev(w, rows, dev.put(xq), dev.put(xs), out)
    want, tol = product(xq, xs, lev, sc, gs)
    got = dev.get(out, (rows, n))
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@pytest.mark.gpu
def test_two_contexts_at_the_same_time():
    """Two contexts, each on a stream of its own, with work of both in flight: the results are those of the calls made alone."""
    import gwenedeg_b200 as gw
    rng = np.random.default_rng(21)
    n, k, gs = 640, 2176, 64
    cs = [gw.Context(0, n_attn=1, n_heads=8, n_kv_heads=2, head_dim=128, max_rows=256) for _ in range(2)]
    ds = [Dev(c) for c in cs]
    lev, sc = matrix(rng, n, k, gs)
    ms = [c.q4_new(packed(lev), sc, gs) for c in cs]
    ins = [[rows8(rng, rows, k, gs) for rows in (1, 40, 200)] for _ in cs]
    ptr = [[(d.put(q), d.put(s), d.room((q.shape[0], n), np.float32)) for q, s in i] for d, i in zip(ds, ins)]
    alone = []
    for c, d, m, pp, ii in zip(cs, ds, ms, ptr, ins):
        for (q, s, o), (xq, _) in zip(pp, ii):
            c.mm_q4_dev(m, xq.shape[0], q, s, o)
            alone.append(d.get(o, (xq.shape[0], n)))
    for _ in range(20):
        for j in range(3):
            for c, m, pp, ii in zip(cs, ms, ptr, ins):
                c.mm_q4_dev(m, ii[j][0].shape[0], *pp[j])
    at = 0
    for d, pp, ii in zip(ds, ptr, ins):
        for (q, s, o), (xq, _) in zip(pp, ii):
            assert np.array_equal(d.get(o, (xq.shape[0], n)), alone[at])
            at += 1
    for d, c in zip(ds, cs):
        d.free()
        c.close()


# ---- the norm ---------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim,gs", [(1, 32, 32), (3, 96, 32), (2, 128, 128), (77, 2720, 32), (5, 4096, 64), (64, 4096, 128), (2, 8320, 64), (1, 32768, 128),
                                         (3, 20480, 32), (300, 192, 64)])
@pytest.mark.parametrize("delta", [True, False])
def test_norm_matches_the_definition(ctx, dev, rows, dim, gs, delta):
    rng = np.random.default_rng(rows + dim)
    eps = 1e-6
    x = rng.standard_normal((rows, dim)).astype(np.float32)
    x[:, dim // 3] *= 30.0
    if rows > 2:
        x[2, :gs] = 0.0
    d = (0.3 * rng.standard_normal((rows, dim))).astype(np.float32) if delta else None
    if delta and rows > 2:
        d[2, :gs] = 0.0
    w = (1.0 + 0.2 * rng.standard_normal(dim)).astype(np.float32)
    x2 = x + d if delta else x
    G = dim // gs
    px, pd, pw = dev.put(x), dev.put(d) if delta else None, dev.put(w)
    po, py = dev.room(rows * dim + 64, np.float32, fill=-7.5), dev.room(rows * dim + 64, np.float32, fill=-7.5)
    pq, ps = dev.room(rows * dim + 64, np.int8, fill=99), dev.room(rows * G + 64, np.float32, fill=-7.5)
    ctx.add_norm_quant_dev(rows, dim, gs, px, pd, pw, eps, po, py, pq, ps)
    o, y, q, s = dev.get(po, rows * dim + 64), dev.get(py, rows * dim + 64), dev.get(pq, rows * dim + 64, np.int8), dev.get(ps, rows * G + 64)
    assert (o[rows * dim:] == -7.5).all() and (y[rows * dim:] == -7.5).all() and (q[rows * dim:] == 99).all() and (s[rows * G:] == -7.5).all()
    o, y, q, s = o[:rows * dim].reshape(rows, dim), y[:rows * dim].reshape(rows, dim), q[:rows * dim].reshape(rows, dim), s[:rows * G].reshape(rows, G)
    assert np.array_equal(o, x2)
    lev, top = quantised(x2 * w, gs)
    assert np.array_equal(q, lev)
    inv = 1.0 / np.sqrt((x2.astype(np.float64) ** 2).mean(1, keepdims=True) + eps)
    # the sum of squares: a thread's chain of at most 32 terms, 5 + 32 additions; its error halves in the root; the division by dim, the
    # addition of eps, the root and the reciprocal, then the products: below (69 + 2) / 2 + 5 half steps
    tol = 41 * U
    assert (np.abs(y - x2 * w.astype(np.float64) * inv) <= tol * np.abs(x2 * w.astype(np.float64) * inv)).all()
    want_s = top.astype(np.float64) / 127.0 * inv
    assert (np.abs(s - want_s) <= tol * want_s).all()
    # each output alone, and x in place
    for name in ("x", "y", "q"):
        p2, y2, q2, s2 = dev.put(x), dev.room((rows, dim), np.float32), dev.room((rows, dim), np.int8), dev.room((rows, G), np.float32)
        ctx.add_norm_quant_dev(rows, dim, gs, p2, pd, pw, eps, p2 if name == "x" else None, y2 if name == "y" else None,
                               q2 if name == "q" else None, s2 if name == "q" else None)
        assert np.array_equal(dev.get(p2, (rows, dim)), x2 if name == "x" else x)
        if name == "y":
            assert np.array_equal(dev.get(y2, (rows, dim)), y)
        if name == "q":
            assert np.array_equal(dev.get(q2, (rows, dim), np.int8), q) and np.array_equal(dev.get(s2, (rows, G)), s)


@pytest.mark.gpu
def test_norm_of_zero_rows_and_of_values_that_are_not_finite(ctx, dev):
    dim, gs = 256, 64
    x = np.ones((4, dim), np.float32)
    x[0] = 0.0
    x[1, 70] = np.nan
    x[2, 130] = np.inf
    q, s, y = dev.room((4, dim), np.int8), dev.room((4, 4), np.float32), dev.room((4, dim), np.float32)
    ctx.add_norm_quant_dev(4, dim, gs, dev.put(x), None, dev.put(np.ones(dim, np.float32)), 0.0, None, y, q, s)
    gq, gsx = dev.get(q, (4, dim), np.int8), dev.get(s, (4, 4))
    assert (gq[0] == 0).all()
    assert np.isnan(gsx[1]).all() and not np.isfinite(dev.get(y, (4, dim))[1]).any()
    assert np.isnan(gsx[2, 2])
    assert (gq[3] == 127).all() and np.allclose(gsx[3] * 127.0, 1.0, rtol=1e-6)
    # with eps the zero row is zero
    ctx.add_norm_quant_dev(4, dim, gs, dev.put(x), None, dev.put(np.ones(dim, np.float32)), 1e-6, None, y, q, s)
    assert (dev.get(y, (4, dim))[0] == 0).all() and (dev.get(s, (4, 4))[0] == 0).all()


# ---- refusals ---------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_refusals(ctx, dev):
    import gwenedeg_b200 as gw
    L = ctx.L
    k, gs, n = 128, 64, 64
    lev = packed(np.zeros((n, k), np.int8))
    sc = np.zeros((n, k // gs), np.float16)
    w = ctx.q4_new(lev, sc, gs)
    other = gw.Context(0, n_attn=1, n_heads=8, n_kv_heads=2, head_dim=128, max_rows=4)
    foreign = other.q4_new(lev, sc, gs)
    narrow = ctx.q4_new(packed(np.zeros((n, 64), np.int8)), np.zeros((n, 1), np.float16), gs)
    b = dev.room(4096, np.float32)
    h = C.c_void_p()

    def refused(rc, text):
        assert rc == -1 and text in L.rq_cuda_error(ctx.h).decode(), (rc, L.rq_cuda_error(ctx.h))

    for bad in ((0, k, gs), (n, 0, gs), (n, 100, 64), (n, 256, 256), (n, 48, 16), (-1, k, gs)):
        refused(L.rq_cuda_q4_new_dev(ctx.h, *bad, b, b, C.byref(h)), "q4_new")
        assert not h.value
    refused(L.rq_cuda_q4_new_dev(ctx.h, n, k, gs, None, b, C.byref(h)), "null")
    refused(L.rq_cuda_q4_new_dev(ctx.h, n, k, gs, b + 2, b, C.byref(h)), "aligned")
    for rows in (0, -1, 513):
        refused(L.rq_cuda_mm_q4_dev(ctx.h, w.h, rows, b, b, b), "rows")
        refused(L.rq_cuda_ffn_q4_dev(ctx.h, w.h, w.h, rows, b, b, b, None, None), "rows")
        refused(L.rq_cuda_add_norm_quant_dev(ctx.h, rows, 128, 64, b, None, b, 1e-6, None, b, None, None), "rows")
    refused(L.rq_cuda_mm_q4_dev(ctx.h, None, 1, b, b, b), "null")
    refused(L.rq_cuda_mm_q4_dev(ctx.h, w.h, 1, None, b, b), "null")
    refused(L.rq_cuda_mm_q4_dev(ctx.h, w.h, 1, b, b, None), "null")
    refused(L.rq_cuda_mm_q4_dev(ctx.h, w.h, 1, b + 8, b, b), "aligned")
    refused(L.rq_cuda_mm_q4_dev(ctx.h, w.h, 1, b, b + 2, b), "aligned")
    refused(L.rq_cuda_mm_q4_dev(ctx.h, w.h, 1, b, b, b + 1), "aligned")
    refused(L.rq_cuda_mm_q4_dev(ctx.h, foreign.h, 1, b, b, b), "another context")
    refused(L.rq_cuda_ffn_q4_dev(ctx.h, w.h, narrow.h, 1, b, b, b, None, None), "matrices")
    refused(L.rq_cuda_ffn_q4_dev(ctx.h, w.h, w.h, 1, b, b, None, None, None), "null")
    refused(L.rq_cuda_ffn_q4_dev(ctx.h, w.h, w.h, 1, b, b, b, b, None), "null")
    for dim, g in ((0, 64), (100, 64), (32768 + 128, 128), (256, 256), (48, 16)):
        refused(L.rq_cuda_add_norm_quant_dev(ctx.h, 1, dim, g, b, None, b, 1e-6, None, b, None, None), "groups")
    refused(L.rq_cuda_add_norm_quant_dev(ctx.h, 1, 128, 64, b, None, b, 1e-6, None, None, None, None), "null")
    refused(L.rq_cuda_add_norm_quant_dev(ctx.h, 1, 128, 64, b, None, b, 1e-6, None, None, b, None), "null")
    refused(L.rq_cuda_add_norm_quant_dev(ctx.h, 1, 128, 64, b + 4, None, b, 1e-6, None, b, None, None), "aligned")
    refused(L.rq_cuda_add_norm_quant_dev(ctx.h, 1, 128, 64, b, None, b, float("nan"), None, b, None, None), "eps")
    refused(L.rq_cuda_add_norm_quant_dev(ctx.h, 1, 128, 64, b, None, b, -1.0, None, b, None, None), "eps")
    with pytest.raises(ValueError):
        ctx.q4_new(lev, sc, 32)
    foreign.free()
    other.close()


# ---- graphs, streams --------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_a_captured_run_replays_on_new_inputs():
    """Norm, product, gated product and product captured into two CUDA graphs on a stream of the caller's, replayed in turn on inputs
    that change in between, give the bits of the plain calls."""
    import torch

    import gwenedeg_b200 as gw
    rng = np.random.default_rng(9)
    k, n, gs, eps = 256, 384, 64, 1e-6
    c = gw.Context(0, n_attn=1, n_heads=8, n_kv_heads=2, head_dim=128, max_rows=128)
    mats = [c.q4_new(packed(lev), sc, gs) for lev, sc in (matrix(rng, k, k, gs), matrix(rng, n, k, gs), matrix(rng, n, k, gs), matrix(rng, k, n, gs))]
    st = torch.cuda.Stream()
    c.set_stream(st.cuda_stream)
    w = torch.ones(k, device="cuda")

    def buffers(rows):
        f = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
        return dict(rows=rows, x=f(rows, k), q=f(rows, k, t=torch.int8), s=f(rows, k // gs), a=f(rows, k), hq=f(rows, n, t=torch.int8), hs=f(rows, n // gs), y=f(rows, k))

    def calls(b):
        p = {i: t.data_ptr() for i, t in b.items() if i != "rows"}
        r = b["rows"]
        c.add_norm_quant_dev(r, k, gs, p["x"], None, w.data_ptr(), eps, None, None, p["q"], p["s"])
        c.mm_q4_dev(mats[0], r, p["q"], p["s"], p["a"])
        c.add_norm_quant_dev(r, k, gs, p["x"], p["a"], w.data_ptr(), eps, p["x"], None, p["q"], p["s"])
        c.ffn_q4_dev(mats[1], mats[2], r, p["q"], p["s"], None, p["hq"], p["hs"])
        c.mm_q4_dev(mats[3], r, p["hq"], p["hs"], p["y"])

    sets, graphs = [buffers(1), buffers(100)], []
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        for b in sets:
            calls(b)  # (kernels are loaded before the capture)
        st.synchronize()
        for b in sets:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                calls(b)
            graphs.append(g)
        for turn in range(3):
            inputs = [torch.from_numpy(rng.standard_normal((b["rows"], k)).astype(np.float32)).cuda() for b in sets]
            got = []
            for b, x in zip(sets, inputs):
                b["x"].copy_(x)
            for g in graphs:
                g.replay()
            st.synchronize()
            got = [(b["x"].clone(), b["y"].clone()) for b in sets]
            for b, x, (gx, gy) in zip(sets, inputs, got):
                b["x"].copy_(x)
                b["y"].zero_()
                calls(b)
                st.synchronize()
                assert torch.equal(b["x"], gx) and torch.equal(b["y"], gy) and float(gy.abs().max()) > 0
    del graphs
    c.set_stream(None)
    c.close()


# ---- together ---------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_a_decode_layer_on_the_device(dev_layer, rows):
    dev_layer(rows)


@pytest.fixture
def dev_layer(checker):
    """One decode layer through the library alone: every step's output against the step's definition on the inputs it had."""
    import gwenedeg_b200 as gw
    from gwenedeg_b200 import synth

    def run(rows):
        from tests.helpers import assert_close
        rng = np.random.default_rng(11)
        H, KV, hd, gs, eps = 8, 2, 128, 64, 1e-6
        dim, ff, kvd = 320, 448, KV * hd
        c = gw.Context(0, n_attn=1, n_heads=H, n_kv_heads=KV, head_dim=hd, max_rows=64)
        d = Dev(c)
        ms = {i: matrix(rng, *s, gs) for i, s in dict(q=(H * hd, dim), k=(kvd, dim), v=(kvd, dim), wo=(dim, H * hd), gate=(ff, dim), up=(ff, dim), down=(dim, ff)).items()}
        W = {i: c.q4_new(packed(lev), sc, gs) for i, (lev, sc) in ms.items()}
        lens = [1 + 37 * i % 300 for i in range(rows)]
        seqs = [c.new_seq(n, gw.KV_F16) for n in lens]
        for i, (s, n) in enumerate(zip(seqs, lens)):
            if n > 1:
                s.fill_synthetic(n - 1, 5 + i)
        x = synth.normal(1, (rows, dim))
        w1, w2 = (1.0 + 0.1 * rng.standard_normal((2, dim))).astype(np.float32)
        nq = np.ones(hd, np.float32)
        f = lambda *s: d.room(s, np.float32)  # noqa: E731
        px, q1, s1 = d.put(x), d.room((rows, dim), np.int8), f(rows, dim // gs)
        qr, kr, vr, o = f(rows, H * hd), f(rows, kvd), f(rows, kvd), f(rows, H * hd)
        oq, os_, a = d.room((rows, H * hd), np.int8), f(rows, H * hd // gs), f(rows, dim)
        hq, hs, y, pn = d.room((rows, ff), np.int8), f(rows, ff // gs), f(rows, dim), d.put(nq)
        q2, s2 = d.room((rows, dim), np.int8), f(rows, dim // gs)
        p1, p2 = d.put(w1), d.put(w2)
        c.set_wo_quant(gs, oq, os_)
        c.pass_begin([(s, n - 1, 1) for s, n in zip(seqs, lens)])
        c.add_norm_quant_dev(rows, dim, gs, px, None, p1, eps, None, None, q1, s1)
        for m, out in (("q", qr), ("k", kr), ("v", vr)):
            c.mm_q4_dev(W[m], rows, q1, s1, out)
        qraw = d.get(qr, (rows, H * hd))
        c.qk_norm_rope_store_dev(0, qr, kr, vr, pn, pn, hd, 1e6)
        c.attn_decode_dev(0, qr, o)
        c.mm_q4_dev(W["wo"], rows, oq, os_, a)
        c.add_norm_quant_dev(rows, dim, gs, px, a, p2, eps, px, None, q2, s2)
        c.ffn_q4_dev(W["gate"], W["up"], rows, q2, s2, None, hq, hs)
        c.mm_q4_dev(W["down"], rows, hq, hs, y)
        c.sync()
        c.pass_end()

        def inside(got, xq, xs, m):
            want, tol = product(xq, xs, *ms[m], gs)
            assert (np.abs(got - want) <= tol).all(), m

        lev, top = quantised(x * w1, gs)
        g1, t1 = d.get(q1, (rows, dim), np.int8), d.get(s1, (rows, dim // gs))
        assert np.array_equal(g1, lev)
        inside(qraw, g1, t1, "q")
        inside(d.get(vr, (rows, kvd)), g1, t1, "v")
        qrot = d.get(qr, (rows, H, hd))
        att = d.get(o, (rows, H, hd))
        for i, (s, n) in enumerate(zip(seqs, lens)):
            assert_close(att[i:i + 1], checker.attention(gw.KV_F16, s.read_kv(0, 0), s.read_kv(0, 1), KV, H, hd, qrot[i:i + 1], np.array([n], np.int32)), f"row {i}")
        go, to = d.get(oq, (rows, H * hd), np.int8), d.get(os_, (rows, H * hd // gs))
        inside(d.get(a, (rows, dim)), go, to, "wo")
        x2 = x + d.get(a, (rows, dim))
        assert np.array_equal(d.get(px, (rows, dim)), x2)
        g2, t2 = d.get(q2, (rows, dim), np.int8), d.get(s2, (rows, dim // gs))
        assert np.array_equal(g2, quantised(x2 * w2, gs)[0])
        gg, gt = product(g2, t2, *ms["gate"], gs)
        uu, ut = product(g2, t2, *ms["up"], gs)
        h = gg / (1 + np.exp(-gg)) * uu
        g3, t3 = d.get(hq, (rows, ff), np.int8), d.get(hs, (rows, ff // gs))
        back = g3.reshape(rows, -1, gs) * t3[:, :, None].astype(np.float64)
        # a level stands for values at most half a unit off (the quantiser's 0.49999997 and fp32 add less than 1e-4 of a unit)
        assert (np.abs(back - h.reshape(rows, -1, gs)) <= 0.5001 * t3[:, :, None] + 1e-5 * np.abs(h).max()).all()
        inside(d.get(y, (rows, dim)), g3, t3, "down")
        d.free()
        c.close()

    return run
