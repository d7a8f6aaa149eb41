"""The products around the attention, launched one behind the other: what a kernel may do while the kernel before it still runs,
several host threads at once, and the one order of the sums."""
import ctypes as C
import os
import re
import subprocess
import sys
import threading

import numpy as np
import pytest

from tests.test_q4_products import SLICE, Dev, ctx, dev, matrix, packed, product, quantised, rows8  # noqa: F401  (ctx, dev: fixtures)

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gwenedeg_b200", "csrc")


def source(name):
    """A source file without its comments."""
    txt = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", txt, flags=re.S))


# ---- the one order of the sums ----------------------------------------------------------------------------------------
def fma32(a, b, c):
    """a b + c of fp32 arrays with one rounding.  The product is exact in 64 bits; the sum is rounded to odd there (by its exact
    remainder), which keeps enough for the rounding to 24 bits to be the only one that counts (Boldo and Melquiond 2008)."""
    p, c = a.astype(np.float64) * b.astype(np.float64), c.astype(np.float64)
    s = p + c
    t = s - p
    rest = (p - (s - t)) + (c - t)  # p + c - s, exactly
    bits = s.view(np.int64)
    even = (rest != 0) & (bits & 1 == 0)
    away = (rest > 0) == (s > 0)  # the exact sum is further from zero than s
    return np.where(even, np.where(away, bits + 1, bits - 1), bits).view(np.float64).astype(np.float32)


def in_order(xq, xs, lev, sc, gs):
    """The product in fp32 in the order that rq_cuda.h states, operation for operation."""
    r, k = xq.shape
    n, G = lev.shape[0], k // gs
    D = np.einsum("rgi,ngi->rng", xq.reshape(r, G, gs).astype(np.float64), lev.reshape(n, G, gs).astype(np.float64), optimize=True)
    slices = []
    for s in range(0, G, SLICE // gs):
        p = np.zeros((r, n), np.float32)
        for g in range(s, min(G, s + SLICE // gs)):
            t = (D[:, :, g] * sc[None, :, g].astype(np.float64)).astype(np.float32)  # (exact in 64 bits, rounded once)
            p = fma32(t, np.broadcast_to(xs[:, None, g], t.shape), p)
        slices.append(p)
    y = np.zeros((r, n), np.float32)
    for s in range(0, len(slices), 2):
        y = y + (slices[s] + slices[s + 1] if s + 1 < len(slices) else slices[s])
    return y


def test_the_fused_operation_of_these_tests_is_rounded_once():
    from fractions import Fraction
    rng = np.random.default_rng(0)
    a, b, c = ((rng.standard_normal(4000) * 2.0 ** rng.integers(-14, 14, 4000)).astype(np.float32) for _ in range(3))
    c[:1000] = -(a[:1000].astype(np.float64) * b[:1000]).astype(np.float32)  # cancelled down to the product's own rounding error
    a[1000:2000] = np.float32(1) + a[1000:2000] * np.float32(2.0 ** -30)  # borders: sums half way between two fp32 numbers, and next to them
    c[1000:2000] = np.ldexp(b[1000:2000], 24) * rng.choice([1, -1, 3], 1000).astype(np.float32)
    got = fma32(a, b, c)
    for x, y, z, g in zip(a, b, c, got):
        want = Fraction(float(x)) * Fraction(float(y)) + Fraction(float(z))
        near = abs(Fraction(float(g)) - want)
        lo, hi = np.nextafter(g, np.float32(-np.inf)), np.nextafter(g, np.float32(np.inf))
        others = [abs(Fraction(float(o)) - want) for o in (lo, hi)]
        assert near < min(others) or (near == min(others) and int(g.view(np.int32)) % 2 == 0)


@pytest.mark.parametrize("k,gs", [(2080, 32), (4160, 64), (2176, 128)])
def test_the_stated_order_is_within_the_bound(k, gs):
    rng = np.random.default_rng(k)
    lev, sc = matrix(rng, 24, k, gs)
    xq, xs = rows8(rng, 10, k, gs)
    want, tol = product(xq, xs, lev, sc, gs)
    assert (np.abs(in_order(xq, xs, lev, sc, gs) - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("k,gs", [(96, 32), (544, 32), (2080, 32), (5664, 32), (192, 64), (4160, 64), (13376, 64), (128, 128), (2176, 128), (13440, 128)])
def test_products_have_the_bits_of_the_stated_order(ctx, dev, k, gs):
    """An odd and an even number of slices, a last chunk that is not full, few rows and many, split over a cluster or not."""
    rng = np.random.default_rng(k + gs)
    n, most = 145, 150
    lev, sc = matrix(rng, n, k, gs)
    xq, xs = rows8(rng, most, k, gs)
    want = in_order(xq, xs, lev, sc, gs)
    w = ctx.q4_new(packed(lev), sc, gs)
    q, s, out = dev.put(xq), dev.put(xs), dev.room((most, n), np.float32)
    for rows in (1, 8, 9, 25, 40, 57, 64, 100, most):
        ctx.mm_q4_dev(w, rows, q, s, out)
        assert np.array_equal(dev.get(out, (rows, n)).view(np.uint32), want[:rows].view(np.uint32)), rows


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("k,gs", [(64, 32), (512, 64), (1024, 128), (4096, 128)])
def test_the_sign_of_a_zero_does_not_depend_on_the_other_rows(ctx, dev, k, gs, gated):
    """Scales so small that the products vanish: the sums are zeros, and the same ones in both kernels."""
    n, most = 64, 200
    rng = np.random.default_rng(k)
    lev = rng.integers(-8, 8, (n, k)).astype(np.int8)
    lev[:32] = -1
    w = ctx.q4_new(packed(lev), np.full((n, k // gs), 2.0 ** -20, np.float16), gs)
    xq = np.ones((most, k), np.int8)
    xs = np.full((most, k // gs), 2.0 ** -149, np.float32)
    q, s, out = dev.put(xq), dev.put(xs), dev.room((most, n), np.float32)
    got = []
    for rows in (1, 40, 64, most):
        if gated:
            ctx.ffn_q4_dev(w, w, rows, q, s, out, None, None)
        else:
            ctx.mm_q4_dev(w, rows, q, s, out)
        got.append(dev.get(out, (rows, n)))
        assert (got[-1] == 0).all()
        assert (got[-1].view(np.uint32) == got[0].view(np.uint32)).all(), rows


# ---- the order of the tiles -------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,gs", [(300, 3400, 512, 64), (200, 1552, 1056, 32), (512, 2000, 640, 128), (70, 4700, 2176, 128), (57, 40, 32, 32), (64, 17, 64, 64),
                                         (100, 130, 96, 32), (200, 16, 128, 128)])
def test_products_over_several_bands_of_tiles(ctx, dev, rows, n, k, gs):
    """More outputs than one band of tiles has, with a last band and a last tile that are not full; inputs shorter than a chunk."""
    rng = np.random.default_rng(rows + n)
    lev, sc = matrix(rng, n, k, gs)
    xq, xs = rows8(rng, rows, k, gs)
    w = ctx.q4_new(packed(lev), sc, gs)
    out = dev.room(rows * n + 64, np.float32, fill=-7.5)
    ctx.mm_q4_dev(w, rows, dev.put(xq), dev.put(xs), out)
    got = dev.get(out, rows * n + 64)
    assert (got[rows * n:] == -7.5).all()
    assert np.array_equal(got[:rows * n].reshape(rows, n).view(np.uint32), in_order(xq, xs, lev, sc, gs).view(np.uint32))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,gs", [(300, 1728, 512, 64), (200, 1664, 1152, 128), (260, 2432, 256, 128), (130, 1600, 544, 32), (60, 128, 128, 128), (57, 32, 32, 32)])
def test_gated_products_over_several_bands_of_tiles(ctx, dev, rows, n, k, gs):
    """The same for the gated product with its rows in 8 bits; groups of 128 outputs lie across two tiles of a pair."""
    rng = np.random.default_rng(rows + n)
    ms = [matrix(rng, n, k, gs) for _ in range(2)]
    xq, xs = rows8(rng, rows, k, gs)
    xs *= np.float32(0.3)
    gate, up = (ctx.q4_new(packed(lev), sc, gs) for lev, sc in ms)
    q, s = dev.put(xq), dev.put(xs)
    h, hq, hs = dev.room((rows, n), np.float32), dev.room(rows * n + 64, np.int8, fill=99), dev.room(rows * (n // gs) + 64, np.float32, fill=-7.5)
    ctx.ffn_q4_dev(gate, up, rows, q, s, h, hq, hs)
    got, lev, sc = dev.get(h, (rows, n)), dev.get(hq, rows * n + 64, np.int8), dev.get(hs, rows * (n // gs) + 64)
    assert (lev[rows * n:] == 99).all() and (sc[rows * (n // gs):] == -7.5).all()
    g, u = (in_order(xq, xs, *m, gs).astype(np.float64) for m in ms)
    want = g / (1.0 + np.exp(-g)) * u
    # on exactly these g and u: e^-g (2 units in the last place = 4 half steps), 1 + e^-g, the division, the product: 7 half steps
    assert (np.abs(got - want) <= 8 * 2.0 ** -24 * np.abs(want) + 1e-37).all()
    wl, top = quantised(got, gs)
    assert np.array_equal(lev[:rows * n].reshape(rows, n), wl)
    assert np.array_equal(sc[:rows * (n // gs)].reshape(rows, -1), top * np.float32(1.0 / 127.0))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,gs", [(1, 1 << 21, 4224, 64), (70, 1 << 21, 4224, 128), (16384, 70000, 32, 32)])
def test_products_beyond_32_bit_offsets(rows, n, k, gs):
    """More than 2^32 bytes of weights, or of outputs: rows and outputs from the front, the middle and the end against 64 bits."""
    import torch

    import gwenedeg_b200 as gw
    c = gw.Context(0, n_attn=1, n_heads=8, n_kv_heads=2, head_dim=128, max_rows=rows)
    gen = torch.Generator(device="cuda").manual_seed(n + rows)
    lev = torch.randint(0, 256, (n, k // 2), generator=gen, dtype=torch.uint8, device="cuda")
    sc = (torch.rand(n, k // gs, generator=gen, device="cuda") * 0.008 + 0.002).half()
    xq = torch.randint(-127, 128, (rows, k), generator=gen, dtype=torch.int8, device="cuda")
    xs = torch.rand(rows, k // gs, generator=gen, device="cuda") * 0.05 + 0.001
    out = torch.empty(rows, n, device="cuda")
    torch.cuda.synchronize()
    w = c.q4_new_dev(n, k, gs, lev.data_ptr(), sc.data_ptr())
    c.mm_q4_dev(w, rows, xq.data_ptr(), xs.data_ptr(), out.data_ptr())
    c.sync()
    rs = sorted({0, rows // 2, rows - 1})
    fs = torch.cat([torch.arange(a, min(n, a + 40)) for a in (0, n // 2 - 7, n - 40)]).cuda()
    levels = torch.stack((lev[fs] & 15, lev[fs] >> 4), 2).view(len(fs), k).to(torch.int8).cpu().numpy() - 8
    want, tol = product(xq[rs].cpu().numpy(), xs[rs].cpu().numpy(), levels, sc[fs].cpu().numpy(), gs)
    got = out[rs][:, fs].cpu().numpy()
    assert (np.abs(got - want) <= tol).all()
    w.free()
    c.close()


# ---- the plan of the products with many rows --------------------------------------------------------------------------
@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """The library's own choice of tile and split, built for the host: (rows, n, k, gs, gated, quant) -> rt, c, p, np, lst, smem."""
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text('#include "q4_plan.h"\nextern "C" void plan(int rows, int tiles, int slices, int gs, int gated, int quant, int n_sm, int *o) {\n'
                                '  const rq::Q4Plan p = rq::q4_plan(rows, tiles, slices, gs, gated, quant, n_sm);\n'
                                '  const int v[6] = {p.rt, p.c, p.p, p.np, p.lst, p.smem};\n  for (int i = 0; i < 6; i++) o[i] = v[i];\n}\n')
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, str(d / "plan.cpp"), "-o", str(d / "plan.so")])
    lib = C.CDLL(str(d / "plan.so"))

    def run(rows, n, k, gs, gated=False, quant=False, n_sm=148):
        o = (C.c_int * 6)()
        lib.plan(rows, -(-n // 16), -(-k // 512), gs, int(gated), int(quant), n_sm, o)
        return dict(zip(("rt", "c", "p", "np", "lst", "smem"), o))

    return run


@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("gated,quant", [(False, False), (True, False), (True, True)])
def test_every_plan_fits_its_shared_memory(plan, gs, gated, quant):
    """Up to the longest inputs that a matrix may have: the pairs of slices cover the inputs, no CTA of a split is without one, and the
    shared memory holds what the kernel puts there, counted here in exact integers."""
    for k in [32, 512, 544, 1024, 1056, 4096, 12288, 25600, 131072] + [1 << b for b in range(18, 31)] + [(1 << 30) - 128, 3 << 27, 130154496, 260309 * 1024]:
        k = max(gs, k // gs * gs)
        for n in (128, 4096, 65536, 1 << 21):
            for rows in (57, 64, 300, 2048, 16384):
                p = plan(rows, n, k, gs, gated, quant)
                pairs = -(-(-(-k // 512)) // 2)
                assert p["rt"] in (32, 64, 128) and 1 <= p["c"] * p["p"] <= 8 and p["lst"] in (1, 2), (k, n, rows, p)
                assert (p["c"] - 1) * p["np"] < pairs <= p["c"] * p["np"], (k, n, rows, p)
                need = 1024 + ((16384 + 128 * p["rt"]) << p["lst"]) + 2 * (512 // gs) * (p["rt"] + 128) * 4 + p["rt"] * 132 * 4 * (p["np"] if p["c"] > 1 else 1)
                assert p["smem"] == need <= 226 * 1024, (k, n, rows, p)
                assert p["p"] == (2 if gated and quant and gs == 128 else 1)


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


def test_attention_behind_a_product_waits_for_it_in_full():
    """The attention and DeltaNet kernels read rows through the read-only path, so their first launch behind a kernel that lets the next
    one start ahead of its own wait is an ordinary one."""
    code = source("rq_cuda.cu")
    for launch in ("= launch_attn_part_tc(t,", "= launch_attn_part<KV_F16>(", "launch_pdl(kv_dequant_f16_kernel<", "= launch_dn_chunk(a,"):
        body = code[:code.index(launch)]
        body = body[body.rindex("\n}\n"):]  # the function's part in front of the launch
        assert "behind_early(c);" in body, launch
        rest = code[code.index(launch):]
        assert "c->early = false;" in rest[:rest.index("c->launches")], launch
    helper = code[code.index("static void behind_early"):]
    assert "early = " not in helper[:helper.index("}")].replace("in_order = c->early", "")  # (a call that fails before its launch leaves it to the next)
    for entry in ("rq_cuda_add_norm_quant_dev", "rq_cuda_mm_q4_dev", "rq_cuda_ffn_q4_dev"):
        body = code[code.index("int " + entry):]
        assert "c->early = true;" in body[:body.index("\n}\n")], entry


@pytest.mark.gpu
@pytest.mark.parametrize("kv,prefill", [("f16", False), ("q8", False), ("q4", False), ("f16", True), ("q8", True)])
def test_attention_right_behind_the_product_that_makes_its_queries(kv, prefill):
    """Query rows written and read again and again with other values, no cache store and no wait in between: the bits of calls that are
    waited for."""
    import gwenedeg_b200 as gw
    rng = np.random.default_rng(31)
    H, hd, k, gs, ctx_len, turns = 8, 128, 256, 64, 600, 8
    rows = 64 if prefill else 5
    c = gw.Context(0, n_attn=1, n_heads=H, n_kv_heads=2, head_dim=hd, max_rows=64)
    d = Dev(c)
    lev, sc = matrix(rng, H * hd, k, gs)
    w = c.q4_new(packed(lev), sc, gs)
    kvt = dict(f16=gw.KV_F16, q8=gw.KV_Q8, q4=gw.KV_Q4)[kv]
    seqs = [c.new_seq(ctx_len + 64, kvt) for _ in range(1 if prefill else rows)]
    for i, s in enumerate(seqs):
        s.fill_synthetic(ctx_len + (64 if prefill else 1), 3 + i)
    ins = [tuple(d.put(a) for a in rows8(rng, rows, k, gs)) for _ in range(turns)]
    q, outs = d.room((rows, H * hd), np.float32), [d.room((rows, H * hd), np.float32) for _ in range(turns)]
    c.pass_begin([(s, ctx_len, 64 if prefill else 1) for s in seqs])
    attend = c.attn_prefill_dev if prefill else c.attn_decode_dev
    alone = []
    for (xq, xs), o in zip(ins, outs):
        c.mm_q4_dev(w, rows, xq, xs, q)
        c.sync()
        attend(0, q, o)
        alone.append(d.get(o, (rows, H * hd)))
    assert not np.array_equal(alone[0], alone[1])
    for _ in range(10):
        for (xq, xs), o in zip(ins, outs):
            c.mm_q4_dev(w, rows, xq, xs, q)
            attend(0, q, o)
    for o, a in zip(outs, alone):
        assert np.array_equal(d.get(o, (rows, H * hd)).view(np.uint32), a.view(np.uint32))
    c.pass_end(commit=False)
    d.free()
    c.close()


# ---- several host threads ---------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows,ks", [(64, (20480, 512, 12288)), (1, (12288, 6656, 5120)), (200, (12288, 4096, 1024))])
@pytest.mark.parametrize("gated", [False, True])
def test_contexts_in_threads_of_their_own(rows, ks, gated):
    """One context per host thread, all on one device, with the same kernels at shapes that want different amounts of shared memory:
    no call is refused and the results are those of the calls made alone."""
    import gwenedeg_b200 as gw
    rng = np.random.default_rng(rows)
    n, gs, turns = 256, 64, 400
    jobs = []
    for k in ks:
        c = gw.Context(0, n_attn=1, n_heads=8, n_kv_heads=2, head_dim=128, max_rows=256)
        d = Dev(c)
        m = [c.q4_new(packed(lev), sc, gs) for lev, sc in (matrix(rng, n, k, gs), matrix(rng, n, k, gs))]
        xq, xs = rows8(rng, rows, k, gs)
        q, s, o = d.put(xq), d.put(xs * np.float32(0.1)), d.room((rows, n), np.float32)
        call = (lambda c=c, m=m, q=q, s=s, o=o: c.ffn_q4_dev(m[0], m[1], rows, q, s, o, None, None)) if gated else (lambda c=c, m=m, q=q, s=s, o=o: c.mm_q4_dev(m[0], rows, q, s, o))
        call()
        jobs.append((c, d, call, o, d.get(o, (rows, n))))
    failed, start = [], threading.Barrier(len(jobs))

    def work(c, call):
        start.wait()
        try:
            for _ in range(turns):
                call()
            c.sync()
        except Exception as e:
            failed.append(e)

    ts = [threading.Thread(target=work, args=(c, call)) for c, _, call, _, _ in jobs]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    got = [d.get(o, (rows, n)) for _, d, _, o, _ in jobs]
    for c, d, *_ in jobs:
        d.free()
        c.close()
    assert not failed, failed
    for g, (*_, alone) in zip(got, jobs):
        assert np.array_equal(g.view(np.uint32), alone.view(np.uint32))


FIRST_CALLS = """
import sys, threading
import numpy as np
sys.path.insert(0, sys.argv[1])
import gwenedeg_b200 as gw
rows, n, k, gs, jobs, failed = 64, 128, 512, 64, [], []
for _ in range(8):
    c = gw.Context(0, n_attn=1, n_heads=8, n_kv_heads=2, head_dim=128, max_rows=64)
    m = c.q4_new(np.full((n, k // 2), 0x99, np.uint8), np.ones((n, k // gs), np.float16), gs)
    jobs.append((c, m, c.to_device(np.ones((rows, k), np.int8)), c.to_device(np.ones((rows, k // gs), np.float32)), c.to_device(np.zeros((rows, n), np.float32))))
start = threading.Barrier(len(jobs))
def work(c, m, q, s, o):
    start.wait()
    try:
        c.mm_q4_dev(m, rows, q, s, o)
        c.sync()
    except Exception as e:
        failed.append(e)
ts = [threading.Thread(target=work, args=j) for j in jobs]
[t.start() for t in ts]
[t.join() for t in ts]
assert not failed, failed
for c, m, q, s, o in jobs:
    got = np.empty((rows, n), np.float32)
    c.d2h(got, o)
    c.sync()
    assert (got == k).all()
"""


@pytest.mark.gpu
def test_the_first_calls_of_a_process_in_several_threads():
    """What the library looks up once per process is there for every thread that asks, the first ones at the same time included."""
    for _ in range(2):
        r = subprocess.run([sys.executable, "-c", FIRST_CALLS, os.path.dirname(os.path.dirname(CSRC))], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr[-600:]


# ---- waits that run out -----------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,gs", [(100, 264, 2176, 64), (300, 384, 8192, 128)])
def test_an_expired_wait_is_reported_and_the_context_goes_on(ctx, dev, rows, n, k, gs):
    """With the status word set by a wait that ran out the products give up their own waits early, but end; rq_cuda_sync reports it once."""
    import gwenedeg_b200 as gw
    rng = np.random.default_rng(k)
    ms = [matrix(rng, n, k, gs) for _ in range(2)]
    xq, xs = rows8(rng, rows, k, gs)
    gate, up = (ctx.q4_new(packed(lev), sc, gs) for lev, sc in ms)
    q, s, out = dev.put(xq), dev.put(xs * np.float32(0.1)), dev.room((rows, n), np.float32)
    hq, hs = dev.room((rows, n // gs * gs), np.int8), dev.room((rows, n // gs), np.float32)

    def calls():
        ctx.mm_q4_dev(gate, rows, q, s, out)
        if n % gs == 0:
            ctx.ffn_q4_dev(gate, up, rows, q, s, None, hq, hs)

    def results():
        return dev.get(out, (rows, n)).view(np.uint32), dev.get(hq, (rows, n // gs * gs), np.int8), dev.get(hs, (rows, n // gs)).view(np.uint32)

    calls()
    want = results()
    ctx.check(ctx.L.rq_cuda_selftest_wait_expiry(ctx.h, 1000))
    calls()
    with pytest.raises(gw.RqCudaError) as e:
        ctx.sync()
    assert e.value.code == -4 and "expired" in str(e.value)
    ctx.sync()
    calls()
    for a, b in zip(results(), want):
        assert np.array_equal(a, b)


# ---- groups of very small values --------------------------------------------------------------------------------------
SMALL = [2.0 ** e for e in (-100, -118, -119, -120, -121, -122, -124, -126, -130, -140)]
LEAST = 2.0 ** -119  # what a group's largest magnitude counts as at least (rq_cuda.h)


@pytest.mark.gpu
@pytest.mark.parametrize("gs", [32, 64, 128])
def test_norm_quantises_groups_of_very_small_values(ctx, dev, gs):
    """Groups whose 127 / max is beyond fp32, down to subnormal numbers: levels and scales stand for the values to half a unit of the
    least maximum all the same."""
    rng = np.random.default_rng(gs)
    eps, rows, dim = 1e-6, len(SMALL), 4 * gs
    x = rng.uniform(-1, 1, (rows, dim)).astype(np.float64) * np.array(SMALL)[:, None]
    x[:, ::gs] = np.array(SMALL)[:, None] * np.array([1, -1, 1, -1])  # the largest of each group
    x[:, 3 * gs:] = 0.0
    x = x.astype(np.float32)
    q, s = dev.room((rows, dim), np.int8), dev.room((rows, 4), np.float32)
    ctx.add_norm_quant_dev(rows, dim, gs, dev.put(x), None, dev.put(np.ones(dim, np.float32)), eps, None, None, q, s)
    lev, sc = dev.get(q, (rows, dim), np.int8).reshape(rows, 4, gs), dev.get(s, (rows, 4))
    v = x.astype(np.float64).reshape(rows, 4, gs)
    top = np.maximum(np.abs(v).max(2), LEAST)
    inv = 1.0 / np.sqrt((v ** 2).mean((1, 2)) + eps)
    # half a unit, the quantiser's 0.49999997 for 0.5, and half steps of 127 / max and of the product with a value of at most 127
    assert (np.abs(lev[:, :3] - 127.0 * v[:, :3] / top[:, :3, None]) <= 0.5 + 4 * 127 * 2.0 ** -24).all()
    assert (lev[:, 3] == 0).all() and (sc[:, 3] == 0).all()
    # 1 / 127, the root, the division and three products, each half a step (no sum of squares: eps is all there is)
    want = (top / 127.0 * inv[:, None])[:, :3]
    assert (np.abs(sc[:, :3] - want) <= 8 * 2.0 ** -24 * want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 20, 100])
@pytest.mark.parametrize("gs", [32, 64, 128])
def test_gated_rows_quantise_groups_of_very_small_values(ctx, dev, rows, gs):
    rng = np.random.default_rng(gs + rows)
    n, k = len(SMALL) * 128, 128
    gate, up = (ctx.q4_new(packed(lev), sc, gs) for lev, sc in (matrix(rng, n, k, gs), matrix(rng, n, k, gs)))
    xq, xs = rows8(rng, rows, k, gs)
    # h is about g u / 2 for small g: the rows' scales put it where the quantiser's inverse overflows
    for r in range(rows):
        xs[r] *= np.float32(np.sqrt(SMALL[r % len(SMALL)]))
    h, hq, hs = dev.room((rows, n), np.float32), dev.room((rows, n), np.int8), dev.room((rows, n // gs), np.float32)
    ctx.ffn_q4_dev(gate, up, rows, dev.put(xq), dev.put(xs), h, hq, hs)
    v = dev.get(h, (rows, n)).astype(np.float64).reshape(rows, -1, gs)
    lev, sc = dev.get(hq, (rows, n), np.int8).reshape(rows, -1, gs), dev.get(hs, (rows, n // gs))
    top = np.abs(v).max(2)
    least = np.maximum(top, LEAST)
    assert (np.abs(lev - 127.0 * v / least[:, :, None]) <= 0.5 + 4 * 127 * 2.0 ** -24).all()
    want = np.where(top > 0, least / 127.0, 0.0)  # (the smallest rows may vanish)
    assert (np.abs(sc - want) <= 2 * 2.0 ** -24 * want).all()


@pytest.mark.gpu
def test_a_norm_weight_that_is_no_number_shows_in_the_scale(ctx, dev):
    dim, gs = 256, 64
    w = np.ones(dim, np.float32)
    w[64:128] = np.nan
    q, s = dev.room((2, dim), np.int8), dev.room((2, 4), np.float32)
    ctx.add_norm_quant_dev(2, dim, gs, dev.put(np.ones((2, dim), np.float32)), None, dev.put(w), 1e-6, None, None, q, s)
    sc = dev.get(s, (2, 4))
    assert np.isnan(sc[:, 1]).all() and np.isfinite(sc[:, [0, 2, 3]]).all()
