// Products of 8-bit rows with 4-bit weight matrices, and the gated feed-forward product built on them.
//
//   y[r][f] = sum over groups of GS inputs  xs[r][g] ws[f][g] D,   D = sum over the group of xq[r][k] wq[f][k]   (an exact integer)
//
// xq, xs: the rows as the quantisers of this library leave them (int8 levels, one fp32 scale per group); wq: levels -8 .. 7, ws: f16.
// The sum over groups has one order, whatever kernel runs and however many rows a pass has: inputs are cut into slices of 512, a
// slice's groups are a chain p = fma(round(D ws), xs, p) in ascending order from 0, two adjacent slices are added (the last one may be alone),
// and the pairs are added in ascending order from 0.
// So a row's result does not depend on the other rows of the pass.
#pragma once
#include <atomic>

#include "attn_decode.cuh"
#include "q4_plan.h"
#include "tc05.cuh"

namespace rq {

// A weight matrix on the device.  levels: [tiles][chunks][16 outputs][4 pieces of 16 bytes]; piece t, 32-bit word s holds the inputs
// 32 s + 8 t + 0..7 of the chunk: byte b has input b in its low half and input 4 + b in its high half, as 4-bit two's complement.
// So a lane (output g = lane / 4, t = lane % 4) of a warp finds in its own 16 bytes what mma.m16n8k32 wants from it as the A operand for
// four steps of 32 inputs, the levels of its B operand are 8 adjacent bytes of a row, and a half byte kept in the upper half of a
// byte is the int8 value 16 times the level: a mask, or a shift and a mask, unpacks four levels.
// scales: [tiles][slices][16 outputs][512 / gs] f16.  Outputs and inputs behind the matrix's end are zero levels with zero scales.
struct Q4View {
    const uint4 *levels;
    const __half *scales;
    int n, k, gs, tiles, chunks, slices;
};

typedef CUresult (*Q4EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                               const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

struct Q4Args {
    Q4View w, up;        // the matrix; the gated product's second matrix
    const int8_t *xq;    // [rows][k]
    const float *xs;     // [rows][k / gs]
    int rows;
    float *out;          // [rows][n], or null (gated product)
    int8_t *hq;          // [rows][n] and [rows][n / gs]: the gated product's rows in 8 bits, or null
    float *hs;
};

// mm: out = x W^T;  gated: out = silu(x W^T) (x Up^T).  n_sm: SMs of the device;  enc: the driver's tensor-map encoder;  err: the
// context's status word (waits that ran out)
cudaError_t launch_q4(const Q4Args &a, bool gated, int n_sm, Q4EncodeFn enc, int *err, cudaStream_t stream);
// lays a matrix out: levels [n][k / 2] bytes, input 2 j in the low half of byte j, 2 j + 1 in the high one, level + 8; scales [n][k / gs]
cudaError_t launch_q4_pack(const uint8_t *levels, const __half *scales, const Q4View &v, cudaStream_t stream);

#ifdef RQ_Q4_INSTANTIATE

// one thread per 32-bit word of the layout
__global__ void q4_pack_levels_kernel(const uint8_t *__restrict__ src, int n, int k, int chunks, size_t words, uint32_t *__restrict__ dst) {
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < words; i += (size_t)gridDim.x * blockDim.x) {
        const int s = i & 3, t = (i >> 2) & 3, f = (i >> 4) & 15;
        const size_t tc = i >> 8;
        const int c = (int)(tc % chunks), k0 = c * Q4_CHUNK + 32 * s + 8 * t;
        const size_t out = tc / chunks * Q4_TILE + f;
        uint32_t w = 0;
        if (out < (size_t)n && k0 < k) {
            const uint32_t in = *reinterpret_cast<const uint32_t *>(src + out * (k / 2) + k0 / 2);
#pragma unroll
            for (int j = 0; j < 8; j++) w |= (((in >> (4 * j)) & 15u) ^ 8u) << (j < 4 ? 8 * j : 8 * (j - 4) + 4);
        }
        dst[i] = w;
    }
}
__global__ void q4_pack_scales_kernel(const __half *__restrict__ src, int n, int groups, int slices, int per, size_t count, __half *__restrict__ dst) {
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += (size_t)gridDim.x * blockDim.x) {
        const int g = (int)(i % per), f = (int)(i / per % Q4_TILE);
        const size_t ts = i / per / Q4_TILE;
        const int sl = (int)(ts % slices), grp = sl * per + g;
        const size_t out = ts / slices * Q4_TILE + f;
        dst[i] = out < (size_t)n && grp < groups ? src[out * groups + grp] : __ushort_as_half(0);
    }
}

cudaError_t launch_q4_pack(const uint8_t *levels, const __half *scales, const Q4View &v, cudaStream_t stream) {
    const size_t words = (size_t)v.tiles * v.chunks * 256, count = (size_t)v.tiles * v.slices * Q4_TILE * (Q4_SLICE / v.gs);
    const unsigned blocks = (unsigned)((words + 255) / 256 < 16384 ? (words + 255) / 256 : 16384);
    q4_pack_levels_kernel<<<blocks, 256, 0, stream>>>(levels, v.n, v.k, v.chunks, words, (uint32_t *)v.levels);
    q4_pack_scales_kernel<<<blocks, 256, 0, stream>>>(scales, v.n, v.k / v.gs, v.slices, Q4_SLICE / v.gs, count, (__half *)v.scales);
    return cudaGetLastError();
}

// The rows' scales: written by the kernel before this one, which may still run when this one starts, so they are no constants of this kernel
// (the read-only path may hold a line from before the write, and the compiler may move such a load over pdl_wait)
__device__ __forceinline__ float ld_f32(const float *p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint4 ldg_stream(const uint4 *p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
__device__ __forceinline__ void mma_s8(int *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8_first(int *d, const uint32_t *a, uint32_t b0, uint32_t b1, int c) {  // (d need not be set to c first)
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c));
}
// An int32 sum S plus the bits of 1.5 2^23 are the bits of the float 1.5 2^23 + S, exactly, while |S| < 2^22 (here S = 16 D, as the levels
// sit in the upper halves of their bytes: |S| <= 16 . 128 . 8 . 128 = 2^21).  With M = 1.5 2^23:  fma(M + S, ws, -M ws) = round(S ws): M ws is
// exact (ws has 11 significant bits), so one multiply-add converts, removes the offset and applies the weight's scale, with the one rounding
// of the product.  The factor 16 is carried to the end, where the total is multiplied by 1 / 16 (both exact while 16 |y| is below 2^128).
constexpr int Q4_MAGIC = 0x4B400000;
constexpr float Q4_MAGIC_F = 12582912.0f;

__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(const float *p, uint32_t rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at));
    return v;
}
// h = g sigmoid(g) u
__device__ __forceinline__ float q4_silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// ---- few rows: weights straight from memory into the registers that feed mma.m16n8k32 ------------------------------------
__device__ __forceinline__ void cp_async16(void *dst, const void *src, bool valid) {  // (not valid: zeros, nothing is read)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(void *dst, const void *src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
// A CTA of NW warps computes 16 outputs (gated: of each matrix) of 8 NT rows; warp w takes the slices w, w + NW, ...  Everything a slice
// needs is asked for before its first product: its weights (a ring of one slice of one matrix in registers, 16-byte loads that are contiguous
// over the warp; what comes next, the other matrix or the next slice, is asked for as the ring is used), the weights' scales, and the rows'
// levels and scales (cp.async into the warp's own part of shared memory, rows 544 bytes apart: conflict-free 8-byte reads).  Outputs are M
// of the MMA, rows N.  The slices' partial sums meet in shared memory and are added in order by the threads that own the outputs.
// Bound by the weights' bytes; the weights' loads do not wait for the kernel before this one (they are constant), so they overlap its end.
// Measured: 65536 x 4096 (groups of 64), one row, 25.5 us = 5.6 TB/s; walking over tiles with resident CTAs instead of one CTA per tile took
// 47 us, prefetching a later CTA's weights into the L2 cache 31 us.
constexpr int Q4R_XROW = Q4_SLICE + 32;  // bytes from row to row of a slice's levels
__host__ __device__ constexpr int q4r_warp_bytes(int gs, int nt) { return 8 * nt * (Q4R_XROW + Q4_SLICE / gs * 4); }

// MULTI: more slices than warps;  MOST: threads at most
template <int GS, int NT, bool GATED, bool MULTI, int MOST>
__global__ void __launch_bounds__(MOST, MOST > 256 ? 1 : NT == 1 && GS >= 64 ? 3 : NT <= 2 ? 2 : 1) q4_rows_kernel(const Q4Args a) {
    constexpr int GC = Q4_CHUNK / GS;        // groups per chunk
    constexpr int PER = Q4_SLICE / GS;       // groups per slice
    constexpr int J = GATED ? 2 : 1;         // matrices
    constexpr int FT = 16 * J, FS = FT + 4;  // outputs of the CTA, and their stride in shared memory (conflict-free stores)
    constexpr int R = 8 * NT;
    extern __shared__ __align__(16) uint8_t rows_smem[];  // per warp: levels [R][544], scales [PER][R]; its partial sums [R][FS] over the levels
    const int NW = blockDim.x >> 5, w = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int row0 = blockIdx.y * R, rows = min(a.rows - row0, R);
    const Q4View &W = a.w;
    const int K = W.k, G = K / GS;
    uint8_t *xl = rows_smem + (size_t)w * q4r_warp_bytes(GS, NT);
    float *xsm = reinterpret_cast<float *>(xl + R * Q4R_XROW);
    auto red = [&](int u) { return reinterpret_cast<float *>(rows_smem + (size_t)u * q4r_warp_bytes(GS, NT)); };

    const size_t at_levels = (size_t)blockIdx.x * W.chunks * 64 + lane, at_scales = ((size_t)blockIdx.x * W.slices * Q4_TILE + g) * PER;
    uint4 ring[4][2];
    auto fetch = [&](const Q4View &M, int chunk, int slot) {  // (behind the end: the last chunk's bytes, not used)
        chunk = min(chunk, W.chunks - 1);
#pragma unroll
        for (int h = 0; h < 2; h++) ring[slot][h] = ldg_stream(M.levels + at_levels + (size_t)chunk * 64 + h * 32);
    };
    union Scales {  // of one output in a slice
        uint2 v[PER / 4];
        __half h[PER];
    } ws[2], wn[2];
    auto fetch_ws = [&](const Q4View &M, int sl) {
        sl = min(sl, W.slices - 1);
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < PER / 4; i++) wn[h].v[i] = __ldg(reinterpret_cast<const uint2 *>(M.scales + at_scales + ((size_t)sl * Q4_TILE + 8 * h) * PER) + i);
    };
    // (the weights are written once, when the matrix is made: their loads need not wait for the kernel before this one)
#pragma unroll
    for (int c = 0; c < 4; c++) fetch(a.w, 4 * w + c, c);
    fetch_ws(a.w, w);
    pdl_launch_dependents();
    pdl_wait();

    constexpr int OWN = R * FT / 128 > 0 ? R * FT / 128 : 1;
    float tot[OWN];
#pragma unroll
    for (int i = 0; i < OWN; i++) tot[i] = 0.0f;

    for (int s0 = 0; s0 < (MULTI ? W.slices : 1); s0 += NW) {
        const int sl = s0 + w;
        float p[J][NT][4];  // output g of rows 2 t, 2 t + 1; output g + 8 of the same
#pragma unroll
        for (int m = 0; m < J; m++)
#pragma unroll
            for (int j = 0; j < NT; j++) p[m][j][0] = p[m][j][1] = p[m][j][2] = p[m][j][3] = 0.0f;
        if (s0 > 0) __syncthreads();  // the last round's partial sums have been read
        if (sl < W.slices) {
            const int k0 = sl * Q4_SLICE + 16 * lane;
#pragma unroll
            for (int r = 0; r < R; r++)
                if (r < rows) cp_async16(xl + r * Q4R_XROW + 16 * lane, a.xq + (size_t)(row0 + r) * K + min(k0, K - 16), k0 < K);
#pragma unroll
            for (int i = 0; i < R * PER / 32; i++) {
                const int e = 32 * i + lane, r = e / PER, gr = sl * PER + e % PER;
                if (r < rows) cp_async4(xsm + (e % PER) * R + r, a.xs + (size_t)(row0 + r) * G + min(gr, G - 1), gr < G);
            }
            if (s0 > 0) fetch_ws(a.w, sl);
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
#pragma unroll
            for (int m = 0; m < J; m++) {
#pragma unroll
                for (int h = 0; h < 2; h++) ws[h] = wn[h];
                if (m + 1 < J) fetch_ws(a.up, sl);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    // (a chunk at a time: without this the compiler unpacks and converts everything ahead and runs out of registers)
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        asm volatile("" : "+r"(ring[c][h].x), "+r"(ring[c][h].y), "+r"(ring[c][h].z), "+r"(ring[c][h].w)::"memory");
#pragma unroll
                    for (int i = 0; i < PER / 2; i++) asm volatile("" : "+r"(ws[i & 1].v[i >> 1].x), "+r"(ws[i & 1].v[i >> 1].y));
                    if (4 * sl + c < W.chunks) {
#pragma unroll
                        for (int gc = 0; gc < GC; gc++) {
                            uint32_t A[GS / 32][4];
                            float wf[2], of[2];
#pragma unroll
                            for (int st = 0; st < GS / 32; st++) {
                                const int s = gc * (GS / 32) + st;
                                const uint32_t lo = s == 0 ? ring[c][0].x : s == 1 ? ring[c][0].y : s == 2 ? ring[c][0].z : ring[c][0].w;
                                const uint32_t hi = s == 0 ? ring[c][1].x : s == 1 ? ring[c][1].y : s == 2 ? ring[c][1].z : ring[c][1].w;
                                A[st][0] = (lo << 4) & 0xF0F0F0F0u;
                                A[st][1] = (hi << 4) & 0xF0F0F0F0u;
                                A[st][2] = lo & 0xF0F0F0F0u;
                                A[st][3] = hi & 0xF0F0F0F0u;
                            }
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                wf[h] = __half2float(ws[h].h[c * GC + gc]);
                                of[h] = -Q4_MAGIC_F * wf[h];
                            }
#pragma unroll
                            for (int j = 0; j < NT; j++) {
                                int d[4];
#pragma unroll
                                for (int st = 0; st < GS / 32; st++) {
                                    const uint2 b = *reinterpret_cast<const uint2 *>(xl + (8 * j + g) * Q4R_XROW + (c * GC + gc) * GS + 32 * st + 8 * t);
                                    if (st == 0) mma_s8_first(d, A[st], b.x, b.y, Q4_MAGIC);
                                    else mma_s8(d, A[st], b.x, b.y);
                                }
                                const float2 x = *reinterpret_cast<const float2 *>(xsm + (c * GC + gc) * R + 8 * j + 2 * t);
#pragma unroll
                                for (int h = 0; h < 2; h++) {
                                    p[m][j][2 * h] = fmaf(fmaf(__int_as_float(d[2 * h]), wf[h], of[h]), x.x, p[m][j][2 * h]);
                                    p[m][j][2 * h + 1] = fmaf(fmaf(__int_as_float(d[2 * h + 1]), wf[h], of[h]), x.y, p[m][j][2 * h + 1]);
                                }
                            }
                        }
                    }
                    if (m + 1 < J) fetch(a.up, 4 * sl + c, c);
                    else if constexpr (MULTI) fetch(a.w, 4 * (sl + NW) + c, c);
                }
            }
            __syncwarp();  // (the partial sums go where the levels were)
        }
#pragma unroll
        for (int m = 0; m < J; m++)
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float *o = red(w) + (8 * j + 2 * t) * FS + 16 * m + 8 * h + g;
                    o[0] = p[m][j][2 * h];
                    o[FS] = p[m][j][2 * h + 1];
                }
        __syncthreads();
        const int nw = min(NW, W.slices - s0);
#pragma unroll
        for (int i = 0; i < OWN; i++) {
            const int e = i * blockDim.x + threadIdx.x;
            if (e < R * FT)
                for (int u = 0; u < nw; u += 2) {
                    const int at = e / FT * FS + e % FT;
                    tot[i] += u + 1 < nw ? red(u)[at] + red(u + 1)[at] : red(u)[at];
                }
        }
    }
    if constexpr (!GATED) {
#pragma unroll
        for (int i = 0; i < OWN; i++) {
            const int e = i * blockDim.x + threadIdx.x, r = e / FT;
            const int f = blockIdx.x * FT + e % FT;
            if (e < R * FT && r < rows && f < W.n) a.out[(size_t)(row0 + r) * W.n + f] = tot[i] * 0.0625f;
        }
    } else {
        // the two products of an output are in different threads: through shared memory
        __syncthreads();
#pragma unroll
        for (int i = 0; i < OWN; i++) {
            const int e = i * blockDim.x + threadIdx.x;
            if (e < R * FT) red(0)[e / FT * FS + e % FT] = tot[i] * 0.0625f;
        }
        __syncthreads();
        float *sum = red(0), *h = sum + R * FS, *top = h + R * 16;  // [R][FS], [R][16], [R]
        for (int e = threadIdx.x; e < R * 16; e += blockDim.x) {
            const int r = e >> 4, fo = e & 15, f = blockIdx.x * 16 + fo;
            const float v = q4_silu_mul(sum[r * FS + fo], sum[r * FS + 16 + fo]);
            if (a.out && r < rows && f < W.n) a.out[(size_t)(row0 + r) * W.n + f] = v;
            if (a.hq) {
                float m = fabsf(v);
#pragma unroll
                for (int o = 8; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                h[e] = v;
                if (fo == 0) top[r] = m;
            }
        }
        if (a.hq) {
            // a group of GS outputs is spread over the GS / 16 CTAs of a cluster: they exchange their maxima
            constexpr int CL = GS / 16;
            cluster_sync_all();
            for (int e = threadIdx.x; e < R * 16; e += blockDim.x) {
                const int r = e >> 4, fo = e & 15;
                float m = 0.0f;
#pragma unroll
                for (int q = 0; q < CL; q++) m = fmaxf(m, ld_cluster(top + r, q));
                if (r < rows) {
                    const size_t f = (size_t)blockIdx.x * 16 + fo;
                    a.hq[(size_t)(row0 + r) * W.n + f] = wo_quant_level(h[e], quant_top(m));
                    if (f % GS == 0) a.hs[(size_t)(row0 + r) * (W.n / GS) + f / GS] = quant_scale(m);
                }
            }
            cluster_sync_all();  // (no CTA leaves while another may still read its maxima)
        }
    }
}

template <int GS, int NT, bool GATED>
cudaError_t launch_q4_rows(const Q4Args &a, cudaStream_t stream) {
    // A warp per slice up to 24 of them where the registers allow it (groups of 64 or 128, 8 rows), up to 8 else; at least four warps own the
    // outputs of the CTA
    constexpr bool WIDE = NT == 1 && GS >= 64;
    const bool wide = WIDE && a.w.slices > 8 && a.w.slices <= 24;
    const int NW = wide ? (a.w.slices + 1) / 2 * 2 : a.w.slices >= 8 ? 8 : 4;
    const size_t smem = (size_t)NW * q4r_warp_bytes(GS, NT);
    auto kern = a.w.slices > NW ? q4_rows_kernel<GS, NT, GATED, true, 256> : q4_rows_kernel<GS, NT, GATED, false, 256>;
    if constexpr (WIDE)
        if (wide) kern = q4_rows_kernel<GS, NT, GATED, false, 768>;
    // (the most that any shape asks of this kernel, not what this one does: the value belongs to the kernel, and another thread's call may be
    // between its own setting and its launch)
    const int most = (WIDE && wide ? 24 : 8) * q4r_warp_bytes(GS, NT);
    if (most > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.w.tiles, (a.rows + 8 * NT - 1) / (8 * NT));
    cfg.blockDim = dim3(32 * NW);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (GATED && a.hq) {
        at[1].id = cudaLaunchAttributeClusterDimension;
        at[1].val.clusterDim.x = GS / 16;
        at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    return cudaLaunchKernelEx(&cfg, kern, a);
}

// ---- many rows: the integer tensor cores --------------------------------------------------------------------------------
// A CTA computes 128 outputs (gated: 64 of each matrix) of RT rows over a range of inputs: D [128 outputs x RT rows] (int32, TMEM) =
// W (int8, 128 inputs per stage) x^T by tcgen05.mma kind::i8, one product per group of GS inputs, exact.  Roles:
//   warps 0 .. 7    drain: a warp owns 32 outputs x RT / 2 rows in accumulator-fragment layout (4 outputs per thread: a scale read from
//                   shared memory serves several values): p = fma(D ws, xs, p), packed over row pairs; the scales are staged by
//                   these warps a slice ahead; the first slice of a pair rests in TMEM
//   4 or 8 warps    unpack: a quarter of a chunk each, 1 KB of a tile per load, straight from the layout (registers, four steps ahead), to
//                   int8 rows of 128 inputs with the 128-byte swizzle (K-major A operand); the warp of a chunk's first quarter also asks
//                   for the rows' levels by TMA (K-major B operand)
//   one warp        issues the MMAs into two D buffers in turn, of as many groups as fill 128 columns (up to a chunk's)
// What bounds it is the drain and what runs beside it.  Fitted over shapes, a chunk of 128 inputs of a 128 x 128 tile takes 650 clocks, whatever its
// groups, and 960 per group, against 256 for its products (tensor pipe 10 % busy with groups of 64, 16 % with groups of 128).  A group's drain
// is one logic operation and two multiply-adds per D value and its part of the loads, about 1,900 warp instructions, of which 512 are packed
// multiply-adds on a pipe that takes one every two clocks; alone it takes 474 clocks.  The rest is not separated by a measurement: the unpack warps
// on the same schedulers and the latencies of TMEM and shared memory, with two drain warps per scheduler and half of the issue slots empty.
// Measured: 2000 x 6144 x 4096 270 us with groups of 64, 512 x 4096 x 12288 81.5 us with groups of 128 (632 TOP/s).  16 drain warps, TMEM loads ahead of their
// use, and three buffers brought nothing; integer conversions instead of the offset cost 15 %, additions of the offset (which the compiler
// puts on the multiply-add pipe) 5 %, three unpack warps instead of eight at 32 and 64 rows 40 %.
// With few tiles the inputs are split over the C CTAs of a cluster at multiples of 1,024: every CTA leaves the sums of its pairs of slices
// in its shared memory and each CTA adds up its share of the rows in the one order, reading from the others'.
constexpr int Q4T_DRAIN = 8, Q4T_BAND = 12;
__host__ __device__ constexpr int q4t_unpack(int rt) { return rt == 128 ? 4 : 8; }  // unpack warps
__host__ __device__ constexpr int q4t_threads(int rt) { return 32 * (Q4T_DRAIN + q4t_unpack(rt) + 4); }  // (the MMA warp's warpgroup has three idle warps)

// The registers of a warpgroup: the drain gets what the others do not need.  Per SM: 32 rows or 64 a tile, 20 warps of 96 at launch: 8 x 128 + 8 x 88 +
// 4 x 40 = 1,888 of 1,920; 128 rows, 16 warps of 128: 8 x 184 + 4 x 96 + 4 x 40 = 2,016 of 2,048 (times 32).  Two things rest on the numbers at launch
// (61,440 or 65,536 registers a CTA), which launch_q4_tiles therefore checks: the split has to fit, or the drain waits for registers for ever;
// and no two of these CTAs fit an SM, so that CTAs of two clusters cannot each wait for the TMEM that the other's holds.
__host__ __device__ constexpr int q4t_launch_regs(int rt) { return rt == 128 ? 128 : 96; }
__host__ __device__ constexpr int q4t_drain_regs(int rt) { return rt == 128 ? 184 : 128; }
__host__ __device__ constexpr int q4t_unpack_regs(int rt) { return rt == 128 ? 96 : 88; }
constexpr int Q4T_ISSUE_REGS = 40;
template <int N>
__device__ __forceinline__ void setmaxnreg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void setmaxnreg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// whether a phase is complete, without waiting
__device__ __forceinline__ bool mbar_try_now(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ void ldg_stream8(const void *p, uint32_t *r) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p));
}
// Two adjacent rows of one output, as the halves of 64-bit registers (float2 values would be taken apart and put together again by moves)
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
// p += round(16 D ws) xs for both rows, from the int32 sums d0, d1 (16 D); w2 = ws twice, o2 = -Q4_MAGIC_F w2.  The offset goes in by one
// logic operation, (d & 0x7fffff) ^ 0x4B400000 (the sums fit 23 bits; flipping their sign bit adds 2^22): additions would be put on the pipe that
// the multiply-adds need (a sixth of the drain's time alone).
__device__ __forceinline__ void q4_add2(uint64_t &p, uint32_t d0, uint32_t d1, uint64_t w2, uint64_t o2, uint64_t x2) {
    asm("{\n.reg .b32 a, b;\n.reg .b64 t;\nlop3.b32 a, %1, %6, %7, 0x6a;\nlop3.b32 b, %2, %6, %7, 0x6a;\nmov.b64 t, {a, b};\nfma.rn.f32x2 t, t, %3, %4;\nfma.rn.f32x2 %0, t, %5, %0;\n}"
        : "+l"(p)
        : "r"(d0), "r"(d1), "l"(w2), "l"(o2), "l"(x2), "r"(0x7fffffu), "r"(Q4_MAGIC));
}

// lst: log2 of the operand stages; np: pairs of slices per CTA (C > 1: also the number of sums kept); clusters of C P CTAs
template <int GS, int RT, bool GATED>
__global__ void __launch_bounds__(q4t_threads(RT), 1)
    q4_tiles_kernel(const Q4Args a, const __grid_constant__ CUtensorMap xmap, const int lst, const int np, const int C, const int P, int *err) {
    constexpr int DW = Q4T_DRAIN, UW = q4t_unpack(RT), GC = Q4_CHUNK / GS, PER = Q4_SLICE / GS, RC = 4 * RT / DW, TILES = GATED ? 4 : 8;
    constexpr int GB = GC < 128 / RT ? GC : 128 / RT, NB = GC / GB;  // groups per D buffer, buffers' worth per chunk
    constexpr int UC = RC < 32 ? RC : 32, NU = UC / 8;  // rows drained at a time
    constexpr int HOLD = 256, TOTAL = HOLD + RT;  // TMEM: two D buffers of 128 columns, a slice's p, the running total
    constexpr int XE = (RT * PER + 32 * DW - 1) / (32 * DW);
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float *xss = reinterpret_cast<float *>(sm + (q4t_stage(RT) << lst));  // [2][PER][RT]
    float *wss = xss + 2 * PER * RT;                                     // [2][PER][128]
    float *sums = wss + 2 * PER * 128;                               // [C > 1 ? np : 1][RT][132]
    __shared__ __align__(8) uint64_t full[4], empty[4], dfull[2], dempty[2], done;
    __shared__ uint32_t tmem_slot;
    __shared__ float top[RT];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Q4View &W = a.w;
    const int K = W.k, G = K / GS;
    // a cluster is P adjacent tiles of C CTAs each along the inputs
    const int kc = blockIdx.x % C, py = blockIdx.x / C % P, index = blockIdx.x / (C * P) * P + py;
    // blocks in bands of Q4T_BAND output tiles, inside a band row tile by row tile: CTAs that run together share both operands' tiles evenly
    const int fts = (W.tiles + TILES - 1) / TILES, rts = (a.rows + RT - 1) / RT;
    const int band = index / (Q4T_BAND * rts), in = index - band * Q4T_BAND * rts, wide = min(Q4T_BAND, fts - band * Q4T_BAND);
    const int ft = band * Q4T_BAND + in % wide, row0 = in / wide * RT;
    const int chunk0 = kc * np * (Q4_PAIR / Q4_CHUNK), chunk1 = min(W.chunks, chunk0 + np * (Q4_PAIR / Q4_CHUNK));
    auto tile_of = [&](int tl) { return min(ft * TILES + (GATED ? tl & 3 : tl), W.tiles - 1); };

    // ---- unpack: warp u takes part u % 4 (tiles 2 part, 2 part + 1) of the chunks u / 4, u / 4 + UW / 4, ... of the range
    const int u = warp - DW, part = u & 3, cu = u >> 2, chunks = chunk1 - chunk0;
    constexpr int CU = UW / 4;
    uint32_t ring[4][2][8];
    const uint8_t *lv[2];
    auto fetch = [&](int rel, int slot) {  // (a chunk behind the last: the last one's bytes, not used)
#pragma unroll
        for (int i = 0; i < 2; i++) ldg_stream8(lv[i] + (size_t)min(rel, chunks - 1) * 1024, ring[slot][i]);
    };
    if (u >= 0 && u < UW) {
#pragma unroll
        for (int i = 0; i < 2; i++)
            lv[i] = reinterpret_cast<const uint8_t *>((GATED && part >= 2 ? a.up : a.w).levels) + ((size_t)tile_of(2 * part + i) * W.chunks + chunk0) * 1024 + (lane & 15) * 64 +
                    (lane >> 4) * 32;
        // (the weights are written once, when the matrix is made: their loads need not wait for the kernel before this one)
#pragma unroll
        for (int i = 0; i < 4; i++) fetch(cu + CU * i, i);
    }
    if (tid == 0) {
        for (int i = 0; i < 4; i++) mbar_init(full + i, 5), mbar_init(empty + i, 1);
        for (int i = 0; i < 2; i++) mbar_init(dfull + i, 1), mbar_init(dempty + i, DW);
        mbar_init(&done, 1);
        mbar_fence_init();
    }
    // TMEM is taken after the wait and before the next kernel may start: a CTA that waits for another kernel holds none, and none
    // that starts beside this CTA can take it first, so that no two kernels wait for each other
    pdl_wait();
    if (warp == DW + UW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = tmem_slot;
    pdl_launch_dependents();

    if (warp < DW) {
        setmaxnreg_inc<q4t_drain_regs(RT)>();
        // ---- drain: the warp's 32 outputs x RC rows in accumulator-fragment layout, output 8 k + lane / 4, rows col0 + 8 i + 2 (lane % 4) + 0, 1
        const int quad = warp & 3, col0 = (warp >> 2) * RC, g4 = lane >> 2, t2 = 2 * (lane & 3);
        const uint32_t mine = tbase + ((uint32_t)(quad * 32) << 16) + col0;
        constexpr int NI = RC / 8;
        uint64_t p[4][NI];  // row pairs
        bool ready = false;  // the next D buffer is known to be complete
        const uint64_t minus_magic = pack2(-Q4_MAGIC_F, -Q4_MAGIC_F);
        int buf = 0;
        uint32_t ph = 0;  // the next D buffer and the phase of its barrier
        const int sl0 = chunk0 / 4, sl1 = (chunk1 + 3) / 4;
        // The scales of a slice, a slice ahead: loaded into registers (from clamped addresses, so that nothing waits for the loads before
        // they are stored) and stored to shared memory when the slice before is done.  Rows: element e = (row e / PER, group e % PER);
        // outputs: four groups of one output per thread.
        constexpr int XW = (128 * (PER / 4) + 32 * DW - 1) / (32 * DW), WT = 32 * DW / (PER / 4);
        float xn[XE];
        uint2 wn[XW];
        const int wf = tid / (PER / 4), wp = tid % (PER / 4) * 4;  // outputs wf + WT i (where there are), first of their groups
        const __half *wsrc[XW];
#pragma unroll
        for (int i = 0; i < XW; i++) {
            const int f = min(wf + WT * i, 127);
            wsrc[i] = (GATED && f >= 64 ? a.up : a.w).scales + ((size_t)tile_of(f >> 4) * W.slices * Q4_TILE + (f & 15)) * PER + wp;
        }
        auto fetch_scales = [&](int sl) {
#pragma unroll
            for (int i = 0; i < XE; i++) {
                const int e = i * 32 * DW + tid;
                xn[i] = ld_f32(a.xs + (size_t)min(row0 + e / PER, a.rows - 1) * G + min(sl * PER + e % PER, G - 1));
            }
#pragma unroll
            for (int i = 0; i < XW; i++) wn[i] = __ldg(reinterpret_cast<const uint2 *>(wsrc[i] + (size_t)sl * Q4_TILE * PER));
        };
        auto put_scales = [&](int sl, int slot) {
#pragma unroll
            for (int i = 0; i < XE; i++) {
                const int e = i * 32 * DW + tid;
                if (e < RT * PER) xss[(slot * PER + e % PER) * RT + e / PER] = row0 + e / PER < a.rows && sl * PER + e % PER < G ? xn[i] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < XW; i++)
                if (wf + WT * i < 128) {
                    const float2 lo = __half22float2(*reinterpret_cast<__half2 *>(&wn[i].x)), hi = __half22float2(*reinterpret_cast<__half2 *>(&wn[i].y));
                    float *o = wss + (slot * PER + wp) * 128 + wf + WT * i;
                    o[0] = lo.x, o[128] = lo.y, o[256] = hi.x, o[384] = hi.y;
                }
            asm volatile("bar.sync 1, %0;" ::"n"(32 * DW) : "memory");
        };
        fetch_scales(sl0);
        put_scales(sl0, 0);
        for (int sl = sl0; sl < sl1; sl++) {
            const int slot = (sl - sl0) & 1, bufs = min(4, chunk1 - 4 * sl) * NB;
            if (sl + 1 < sl1) fetch_scales(sl + 1);
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < NI; i++) p[k][i] = 0;
            const float *xsl = xss + slot * PER * RT + col0 + t2, *wsl = wss + slot * PER * 128 + quad * 32 + g4;
#pragma unroll 1
            for (int b = 0; b < bufs; b++) {
                // (asked for ahead: the answer takes ~140 clocks.  After a wait that ran out the loop goes on, with nothing but numbers at stake)
                if (!ready) mbar_wait_bounded_quiet(dfull + buf, ph, err, 82);
                __syncwarp();
                tc_fence_after();
                const uint32_t dbuf = mine + buf * 128;
                uint64_t *const free_bar = dempty + buf;
                buf ^= 1, ph ^= buf == 0;
#pragma unroll
                for (int g = 0; g < GB; g++) {
                    const int at = b * GB + g;
                    uint64_t w2[4], o2[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float w = wsl[at * 128 + 8 * k];
                        w2[k] = pack2(w, w);
                        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(o2[k]) : "l"(w2[k]), "l"(minus_magic));
                    }
#pragma unroll
                    for (int c = 0; c < RC; c += UC) {
                        uint32_t r[2][4 * NU];
#pragma unroll
                        for (int h = 0; h < 2; h++) tmem_ld_frag<NU>(dbuf + ((uint32_t)(16 * h) << 16) + g * RT + c, r[h]);
                        uint64_t x2[NU];
#pragma unroll
                        for (int i = 0; i < NU; i++) x2[i] = *reinterpret_cast<const uint64_t *>(xsl + at * RT + c + 8 * i);
                        tmem_wait_ld();
                        if (g == GB - 1 && c + UC == RC) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(free_bar);
                            ready = mbar_try_now(dfull + buf, ph);
                        }
#pragma unroll
                        for (int i = 0; i < NU; i++)
#pragma unroll
                            for (int k = 0; k < 4; k++) q4_add2(p[k][c / 8 + i], r[k >> 1][4 * i + 2 * (k & 1)], r[k >> 1][4 * i + 2 * (k & 1) + 1], w2[k], o2[k], x2[i]);
                    }
                }
            }
            // the end of the slice: hold p, or add it to the slice before and keep the pair (C > 1) or add it to the total
            constexpr int NE = NI < 4 ? NI : 4;  // pieces of 8 NE rows
            const int pair = (sl - sl0) >> 1;
            const bool hold = !(sl & 1) && sl + 1 < sl1, more = C == 1 && pair > 0, store = !hold && (C > 1 || sl + 1 == sl1);
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int c = 0; c < NI; c += NE) {
                    const uint32_t at = mine + ((uint32_t)(16 * h) << 16) + 8 * c;
                    uint32_t q[4 * NE];
                    auto plus = [&](uint32_t from) {
                        tmem_ld_frag<NE>(from, q);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < NE; i++)
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                uint64_t &v = p[2 * h + k][c + i];
                                asm volatile("{\n.reg .b64 t;\nmov.b64 t, {%1, %2};\nadd.rn.f32x2 %0, t, %0;\n}" : "+l"(v) : "r"(q[4 * i + 2 * k]), "r"(q[4 * i + 2 * k + 1]));
                            }
                    };
                    if (!hold && (sl & 1)) plus(at + HOLD);
                    if (!hold && more) plus(at + TOTAL);
#pragma unroll
                    for (int i = 0; i < NE; i++)
#pragma unroll
                        for (int k = 0; k < 2; k++) q[4 * i + 2 * k] = (uint32_t)p[2 * h + k][c + i], q[4 * i + 2 * k + 1] = (uint32_t)(p[2 * h + k][c + i] >> 32);
                    if (!store) tmem_st_frag<NE>(at + (hold ? HOLD : TOTAL), q);
                    else {
                        float *o = sums + ((size_t)(C > 1 ? pair : 0) * RT + col0 + 8 * c + t2) * Q4T_FS + quad * 32 + 16 * h + g4;
#pragma unroll
                        for (int i = 0; i < 4 * NE; i++) o[(8 * (i >> 2) + (i & 1)) * Q4T_FS + 8 * ((i >> 1) & 1)] = __uint_as_float(q[i]);
                    }
                }
            tmem_wait_st();
            if (sl + 1 < sl1) put_scales(sl + 1, slot ^ 1);
        }
    } else if (u < UW) {
        setmaxnreg_dec<q4t_unpack_regs(RT)>();
        bool ok = true;
        const int f = lane & 15, h = lane >> 4;
        uint8_t *out[4];  // the lane's four 16-byte places in the first tile of its part
#pragma unroll
        for (int s = 0; s < 4; s++) out[s] = sm + part * 4096 + f * 128 + (((2 * s + h) ^ (f & 7)) << 4);
        for (int r0 = cu; r0 < chunks && ok; r0 += 4 * CU) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int rel = r0 + CU * i, st = rel & ((1 << lst) - 1);
                if (rel < chunks && ok) {
                    const int at = st * q4t_stage(RT);
                    if (rel >> lst) ok = mbar_wait_bounded_quiet(empty + st, (uint32_t)((rel >> lst) - 1) & 1u, err, 84);
                    ok = __all_sync(0xffffffffu, ok);
                    if (part == 0 && lane == 0 && ok) {
                        mbar_expect_tx(full + st, RT * 128);
                        tma_load_2d(sm + at + 16384, &xmap, (chunk0 + rel) * Q4_CHUNK, row0, full + st);
                    }
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int s = 0; s < 4; s++) {
                            const uint32_t w0 = ring[i][t][s], w1 = ring[i][t][4 + s];
                            *reinterpret_cast<uint4 *>(out[s] + at + t * 2048) = make_uint4((w0 << 4) & 0xF0F0F0F0u, w0 & 0xF0F0F0F0u, (w1 << 4) & 0xF0F0F0F0u, w1 & 0xF0F0F0F0u);
                        }
                    fetch(rel + 4 * CU, i);
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + st);
                }
            }
        }
        if (lane == 0 && *reinterpret_cast<volatile int *>(err) != 0)  // a wait ran out: the copies in flight get a bounded time to land
            for (int i = 0; i < (1 << lst); i++) mbar_drain(full + i, 0), mbar_drain(full + i, 1);
    } else {
        setmaxnreg_dec<Q4T_ISSUE_REGS>();
        if (u == UW && elect_one()) {
            // ---- MMA issue
            constexpr uint32_t idesc = umma_idesc_i8(128, RT, 0, 0, 1, 1);
            const uint32_t sbase = smem_u32(sm);
            int buf = 0;
            uint32_t ph = 1;  // the phase of the D buffer's barrier before its last release (the first round does not wait)
            bool ok = true;
            for (int chunk = chunk0; chunk < chunk1 && ok; chunk++) {
                const int rel = chunk - chunk0, st = rel & ((1 << lst) - 1);
                ok = mbar_wait_bounded_quiet(full + st, (uint32_t)(rel >> lst) & 1u, err, 85);
                const uint32_t A = sbase + st * q4t_stage(RT), B = A + 16384;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    if (ok && (rel * NB + b >= 2)) ok = mbar_wait_bounded_quiet(dempty + buf, ph, err, 86);
                    if (ok) {
                        tc_fence_after();
#pragma unroll
                        for (int s = 0; s < GB * GS / 32; s++) {
                            const int at = b * GB * GS + 32 * s;
                            umma_i8(tbase + buf * 128 + s / (GS / 32) * RT, umma_desc(A + at, 16, 1024, 2), umma_desc(B + at, 16, 1024, 2), idesc, s % (GS / 32) > 0);
                        }
                        umma_commit(dfull + buf);
                        buf ^= 1, ph ^= buf == 0;
                    }
                }
                umma_commit(empty + st);
            }
            umma_commit(&done);
            mbar_drain(&done, 0);  // (no MMA and no arrival of one is in flight when the CTA ends)
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == DW + UW) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(512));
    if (C > 1) cluster_sync_all();  // (the clusters of 128-wide groups and C = 1 have nothing to read here yet)
    if (warp >= DW) {  // the other roles have only the cluster's barriers left
        if (GATED && a.hq && GS == 128) cluster_sync_all();
        if (C > 1 || P > 1) cluster_sync_all();
        return;
    }

    // ---- the totals of this CTA's share of the rows, a warp per row, lanes along the outputs
    const int share = (RT + C - 1) / C, r0 = kc * share, r1 = min(min(r0 + share, RT), a.rows - row0);
    const int pairs = (W.chunks + 7) / 8;
    const uint32_t prank = (uint32_t)py * C;
    // outputs f, f + 32, f + 64, f + 96 of row r: the pairs' sums in order (the four sums' remote loads overlap)
    auto totals = [&](int r, int f, float *t) {
        if (C == 1) {
#pragma unroll
            for (int i = 0; i < 4; i++) t[i] = (0.0f + sums[r * Q4T_FS + f + 32 * i]) * 0.0625f;  // (from 0: a vanished -0 is 0)
            return;
        }
        t[0] = t[1] = t[2] = t[3] = 0.0f;
#pragma unroll 2
        for (int q = 0; q < pairs; q++) {
            const float *o = sums + ((size_t)(q % np) * RT + r) * Q4T_FS + f;
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = ld_cluster(o + 32 * i, prank + q / np);
#pragma unroll
            for (int i = 0; i < 4; i++) t[i] += v[i];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) t[i] *= 0.0625f;
    };
    if constexpr (!GATED) {
        for (int r = r0 + warp; r < r1; r += DW) {
            float v[4];
            totals(r, lane, v);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int f = ft * 128 + 32 * i + lane;
                if (f < W.n) a.out[(size_t)(row0 + r) * W.n + f] = v[i];
            }
        }
    } else {
        for (int pass = a.hq && GS == 128 ? 0 : 1; pass < 2; pass++) {
            if (pass == 1 && a.hq && GS == 128) cluster_sync_all();  // the two CTAs of a group's halves have their maxima
            for (int r = r0 + warp; r < r1; r += DW) {
                float s[4], v[2];  // gate, gate, up, up
                uint32_t m[2];
                totals(r, lane, s);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    v[i] = q4_silu_mul(s[i], s[2 + i]);
                    m[i] = a.hq ? __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fabsf(v[i]), 0.0f))) : 0u;  // (a NaN counts as 0)
                }
                if (GS >= 64) m[0] = m[1] = max(m[0], m[1]);
                if (pass == 0) {
                    if (lane == 0) top[r] = __uint_as_float(m[0]);
                    continue;
                }
                if (a.hq && GS == 128) {
                    const uint32_t other = (uint32_t)(py ^ 1) * C + kc;
                    m[0] = m[1] = max(m[0], __float_as_uint(ld_cluster(top + r, other)));
                }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int f = ft * 64 + 32 * i + lane;
                    const size_t at = (size_t)(row0 + r) * W.n + f;
                    if (f < W.n) {
                        if (a.out) a.out[at] = v[i];
                        if (a.hq) {
                            a.hq[at] = wo_quant_level(v[i], quant_top(__uint_as_float(m[i])));
                            if (f % GS == 0) a.hs[at / GS] = quant_scale(__uint_as_float(m[i]));
                        }
                    }
                }
            }
        }
    }
    if (C > 1 || P > 1) cluster_sync_all();  // no CTA leaves while another may still read its sums or maxima
}

template <int GS, int RT, bool GATED>
cudaError_t launch_q4_tiles(const Q4Args &a, const Q4Plan &plan, Q4EncodeFn enc, int *err, cudaStream_t stream) {
    const int C = plan.c, P = plan.p;
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)a.w.k, (cuuint64_t)a.rows}, strides[1] = {(cuuint64_t)a.w.k};
    const cuuint32_t box[2] = {Q4_CHUNK, RT}, es[2] = {1, 1};
    if (!enc || enc(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(a.xq), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    auto kern = q4_tiles_kernel<GS, RT, GATED>;
    static_assert(Q4T_DRAIN * q4t_drain_regs(RT) + q4t_unpack(RT) * q4t_unpack_regs(RT) + 4 * Q4T_ISSUE_REGS <= q4t_threads(RT) / 32 * q4t_launch_regs(RT), "split of the registers");
    static_assert(2 * q4t_threads(RT) * q4t_launch_regs(RT) > 65536, "one CTA per SM");
    static std::atomic<bool> checked[64];
    int dev = -1;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !checked[dev]) {
        cudaFuncAttributes fa;
        const cudaError_t e = cudaFuncGetAttributes(&fa, kern);
        if (e != cudaSuccess) return e;
        if (fa.numRegs != q4t_launch_regs(RT)) return cudaErrorInvalidKernelImage;  // (built by another compiler: see q4t_launch_regs)
        if (dev >= 0 && dev < 64) checked[dev] = true;
    }
    // (the same value in every call: it belongs to the kernel, and another thread's call may be between its own setting and its launch)
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Q4T_SMEM);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    const int tiles = GATED ? 4 : 8;
    const int fts = (a.w.tiles + tiles - 1) / tiles, rts = (a.rows + RT - 1) / RT;
    cfg.gridDim = dim3((unsigned)(C * fts * rts));
    cfg.blockDim = dim3(q4t_threads(RT));
    cfg.dynamicSmemBytes = plan.smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = C * P;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = C * P > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, a, map, plan.lst, plan.np, C, P, err);
}

// Up to this many rows the kernel for few rows runs, in blocks of 8 or 16 rows (a block of 16 is counted as 1.75 blocks of 8).  One number for all
// shapes, right for most.  Measured, few rows / many rows in us:
//   rows                           17            32            40            48            56            64
//   6144 x 4096, groups of 32      11.0 / 18.6   13.0 / 18.7   17.5 / 28.6   17.6 / 28.6   21.9 / 28.6   23.7 / 28.7
//   6144 x 4096, 64                 9.7 / 14.9   10.7 / 15.0   14.2 / 19.5   13.7 / 19.5   17.5 / 19.6   18.4 / 19.6
//   4096 x 12288, 64               20.5 / 21.4   20.0 / 22.1   31.5 / 29.1   27.9 / 29.3   35.0 / 29.6   35.8 / 30.1
//   4096 x 12288, 128              19.3 / 19.7   19.5 / 20.5   30.2 / 24.9   27.0 / 25.2   33.3 / 25.5   34.7 / 26.0
//   65536 x 4096, 64               84.6 / 91.2   93.2 / 92.2    157 / 117     139 / 117     179 / 118     186 / 119
//   gated 12288 x 4096, 64, 8-bit  42.0 / 47.5   45.8 / 47.8   67.3 / 63.5   66.1 / 63.5   83.5 / 63.6   84.9 / 63.7
//   gated 12288 x 4096, 128        39.9 / 54.3   43.4 / 54.7   65.6 / 73.4   64.1 / 73.5   83.9 / 73.5   84.3 / 73.6
// So it errs where the many-row kernel has enough tiles for the SMs or long inputs: from 33 rows on 65536 outputs (up to 1.5 x: the blocks of rows
// also read such a matrix from memory once each), from 33 or 49 rows on 12288 inputs and on gated products with groups of 64 (up to 1.3 x).  40
// rows (five blocks of 8) take up to 1.2 x of what 48 rows (three blocks of 16) take: a block of 16 costs less than 1.75 there.
constexpr int Q4_FEW = 56;

template <int GS>
cudaError_t launch_q4_gs(const Q4Args &a, bool gated, int n_sm, Q4EncodeFn enc, int *err, cudaStream_t stream) {
#define Q4_BY_ROWS(GATED_)                                                                  \
    if (a.rows <= Q4_FEW) {                                                                 \
        if (7 * ((a.rows + 15) / 16) > 4 * ((a.rows + 7) / 8)) return launch_q4_rows<GS, 1, GATED_>(a, stream); \
        return launch_q4_rows<GS, 2, GATED_>(a, stream);                                    \
    }                                                                                       \
    const Q4Plan plan = q4_plan(a.rows, a.w.tiles, a.w.slices, GS, GATED_, a.hq != nullptr, n_sm); \
    if (plan.rt == 32) return launch_q4_tiles<GS, 32, GATED_>(a, plan, enc, err, stream); \
    if (plan.rt == 64) return launch_q4_tiles<GS, 64, GATED_>(a, plan, enc, err, stream); \
    return launch_q4_tiles<GS, 128, GATED_>(a, plan, enc, err, stream)
    if (gated) { Q4_BY_ROWS(true); }
    Q4_BY_ROWS(false);
#undef Q4_BY_ROWS
}

cudaError_t launch_q4(const Q4Args &a, bool gated, int n_sm, Q4EncodeFn enc, int *err, cudaStream_t stream) {
    switch (a.w.gs) {
        case 32: return launch_q4_gs<32>(a, gated, n_sm, enc, err, stream);
        case 64: return launch_q4_gs<64>(a, gated, n_sm, enc, err, stream);
        default: return launch_q4_gs<128>(a, gated, n_sm, enc, err, stream);
    }
}

#endif  // RQ_Q4_INSTANTIATE

}  // namespace rq
