// The sizes that the products of 8-bit rows with 4-bit matrices are made of, and the choice of tile and split for many rows.  Plain C++.
#pragma once

#ifdef __CUDACC__
#define RQ_HD __host__ __device__
#else
#define RQ_HD
#endif

namespace rq {

constexpr int Q4_TILE = 16;    // outputs per tile of the layout
constexpr int Q4_CHUNK = 128;  // inputs per chunk: a (tile, chunk) is 1 KB
constexpr int Q4_SLICE = 512;  // inputs per slice of the sum's order
constexpr int Q4_PAIR = 1024;  // ... and per pair of slices

// Shared memory of the kernel for many rows, in bytes: an operand stage, two slices' scales of the rows and of the outputs, one
// pair's sums [rt][132]
constexpr int Q4T_FS = 132;
constexpr int Q4T_SMEM = 226 * 1024;  // a CTA's at most
RQ_HD constexpr int q4t_stage(int rt) { return 16384 + rt * 128; }
RQ_HD constexpr int q4t_scales(int gs, int rt) { return 2 * (Q4_SLICE / gs) * (rt + 128) * 4; }
RQ_HD constexpr int q4t_sums(int rt) { return rt * Q4T_FS * 4; }
// ... beside the stages, with np pairs per CTA (64 bits: a CTA of a long split would hold far more than 2^31)
RQ_HD constexpr long long q4t_fixed(int gs, int rt, int c, int np) { return 1024 + q4t_scales(gs, rt) + (long long)q4t_sums(rt) * (c > 1 ? np : 1); }

struct Q4Plan {
    int rt, c;     // rows per tile; CTAs along the inputs
    int p;         // adjacent tiles per cluster (2: groups of 128 outputs in 8 bits span two gated tiles)
    int np;        // pairs of slices per CTA
    int lst;       // log2 of the operand stages
    int smem;
};
// Rows per tile and CTAs along the inputs with the least estimated time, in clocks.  CTAs run one per SM, in waves; a CTA costs 6,000 to start
// and end (2,500 more in a cluster) and a chunk of 128 inputs a part for its stage and a part per group that is drained, as measured:
// 32 rows 750 + 190, 64 rows 700 + 500, 128 rows 650 + 960.  Fitted to products: 2000 x 6144 x 4096 comes out as 269 us (measured 270), 512 x 4096 x
// 12288 as 81.7 (81.5).  A gated product's epilogue is in no term: 1024 x 12288 x 4096 comes out as 494 us (measured 535).
inline Q4Plan q4_plan(int rows, int w_tiles, int slices, int gs, bool gated, bool quant, int n_sm) {
    const int pairs = (slices + 1) / 2, tiles = (w_tiles + (gated ? 3 : 7)) / (gated ? 4 : 8), p = gated && quant && gs == 128 ? 2 : 1;
    Q4Plan best = {};
    double least = 1e300;
    for (int rt = 32; rt <= 128; rt *= 2) {
        const double chunk = rt == 128 ? 650.0 + 960.0 * (Q4_CHUNK / gs) : rt == 64 ? 700.0 + 500.0 * (Q4_CHUNK / gs) : 750.0 + 190.0 * (Q4_CHUNK / gs);
        for (int c = 1; c * p <= 8 && c <= pairs; c++) {
            const int np = (pairs + c - 1) / c;
            if ((pairs + np - 1) / np != c) continue;
            const long long fixed = q4t_fixed(gs, rt, c, np);
            if (fixed + 2 * q4t_stage(rt) > Q4T_SMEM) continue;
            const long long ctas = (long long)c * tiles * ((rows + rt - 1) / rt), slots = n_sm / (c * p) * (c * p);
            const double time = (double)((ctas + slots - 1) / slots) * (6000.0 + (c > 1 ? 2500.0 : 0.0) + (double)np * (Q4_PAIR / Q4_CHUNK) * chunk);
            const int lst = (Q4T_SMEM - fixed) / q4t_stage(rt) >= 4 ? 2 : 1;
            if (time < least) least = time, best = {rt, c, p, np, lst, (int)(fixed + (q4t_stage(rt) << lst))};
        }
    }
    return best;
}

}  // namespace rq
