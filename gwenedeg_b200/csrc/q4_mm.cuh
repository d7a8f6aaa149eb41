// Products of 8-bit rows with 4-bit weight matrices, and the gated feed-forward product built on them.
//
//   y[r][f] = sum over groups of GS inputs  xs[r][g] ws[f][g] D,   D = sum over the group of xq[r][k] wq[f][k]   (an exact integer)
//
// xq, xs: the rows as the quantisers of this library leave them (int8 levels, one fp32 scale per group); wq: levels -8 .. 7, ws: f16.
// The sum over groups has one order, whatever kernel runs and however many rows a pass has: inputs are cut into slices of 512, a
// slice's groups are a chain p = fma(D, ws xs, p) in ascending order from 0, two adjacent slices are added (the last one may be alone),
// and the pairs are added in ascending order from 0.
// So a row's result does not depend on the other rows of the pass.
#pragma once
#include "attn_decode.cuh"
#include "tc05.cuh"

namespace rq {

constexpr int Q4_TILE = 16;    // outputs per tile of the layout
constexpr int Q4_CHUNK = 128;  // inputs per chunk: a (tile, chunk) is 1 KB
constexpr int Q4_SLICE = 512;  // inputs per slice of the sum's order
constexpr int Q4_PAIR = 1024;  // ... and per pair of slices

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
// An int32 accumulator that starts at the bits of 1.5 2^23 ends as the bits of the float 1.5 2^23 + sum, exactly, while |sum| < 2^22
// (here |16 D| <= 16 . 128 . 8 . 128 = 2^21): one subtraction instead of an integer conversion.
constexpr int Q4_MAGIC = 0x4B400000;
constexpr float Q4_MAGIC_F = 12582912.0f;

// h = g sigmoid(g) u
__device__ __forceinline__ float q4_silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// The simple kernel, right for every size: a CTA of NW warps computes 16 MT outputs (gated: 16 outputs of each matrix) of 8 NT rows, warp
// w takes the slices w, w + NW, ...; weights go from global memory straight into the registers of the lane that feeds them to
// mma.m16n8k32 (outputs as M, rows as N), the rows' levels come through L1.  The slices' partial sums meet in shared memory and are
// added in order by the threads that own the outputs.
template <int GS, int MT, int NT, bool GATED>
__global__ void __launch_bounds__(256) q4_rows_kernel(const Q4Args a) {
    constexpr int GC = Q4_CHUNK / GS;        // groups per chunk
    constexpr int PER = Q4_SLICE / GS;       // groups per slice
    constexpr int FT = 16 * MT, FS = FT + 4;  // outputs of the CTA, and their stride in shared memory (conflict-free stores)
    constexpr int R = 8 * NT;
    extern __shared__ float red[];  // [NW][R][FS]
    const int NW = blockDim.x >> 5, w = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int row0 = blockIdx.y * R, rows = min(a.rows - row0, R);
    const Q4View &W = a.w;
    const int K = W.k, G = K / GS;

    const uint4 *lv[MT];
    const __half *sc[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const Q4View &M = GATED && m == 1 ? a.up : a.w;
        const size_t tile = GATED ? blockIdx.x : min((int)blockIdx.x * MT + m, W.tiles - 1);
        lv[m] = M.levels + tile * W.chunks * 64 + lane;
        sc[m] = M.scales + tile * W.slices * Q4_TILE * PER + g * PER;
    }
    uint4 ring[4][MT][2];
    auto fetch = [&](int chunk, int slot) {
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int h = 0; h < 2; h++)
                ring[slot][m][h] = chunk < W.chunks ? ldg_stream(lv[m] + (size_t)chunk * 64 + h * 32) : make_uint4(0, 0, 0, 0);
    };
    // (the weights are written once, when the matrix is made: their loads need not wait for the kernel before this one)
#pragma unroll
    for (int c = 0; c < 4; c++) fetch(4 * w + c, c);
    pdl_launch_dependents();
    pdl_wait();

    const int8_t *xr[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) xr[j] = a.xq + (size_t)(row0 + min(8 * j + g, rows - 1)) * K + 8 * t;
    float tot[R * FT / 128 > 0 ? R * FT / 128 : 1];
#pragma unroll
    for (int i = 0; i < (int)(sizeof(tot) / 4); i++) tot[i] = 0.0f;

    for (int s0 = 0; s0 < W.slices; s0 += NW) {
        const int sl = s0 + w;
        float p[MT][NT][4];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) p[m][j][i] = 0.0f;
        if (sl < W.slices) {
            const __half *ss[MT];
#pragma unroll
            for (int m = 0; m < MT; m++) ss[m] = sc[m] + (size_t)sl * Q4_TILE * PER;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int chunk = 4 * sl + c;
                if (chunk < W.chunks) {
#pragma unroll
                    for (int gc = 0; gc < GC; gc++) {
                        const int grp = chunk * GC + gc;
                        if (grp < G) {
                            uint32_t A[MT][GS / 32][4];
                            float ws[MT][2];
#pragma unroll
                            for (int m = 0; m < MT; m++) {
#pragma unroll
                                for (int st = 0; st < GS / 32; st++) {
                                    const int s = gc * (GS / 32) + st;
                                    const uint32_t lo = s == 0 ? ring[c][m][0].x : s == 1 ? ring[c][m][0].y : s == 2 ? ring[c][m][0].z : ring[c][m][0].w;
                                    const uint32_t hi = s == 0 ? ring[c][m][1].x : s == 1 ? ring[c][m][1].y : s == 2 ? ring[c][m][1].z : ring[c][m][1].w;
                                    A[m][st][0] = (lo << 4) & 0xF0F0F0F0u;
                                    A[m][st][1] = (hi << 4) & 0xF0F0F0F0u;
                                    A[m][st][2] = lo & 0xF0F0F0F0u;
                                    A[m][st][3] = hi & 0xF0F0F0F0u;
                                }
                                // (1 / 16: the levels are in the upper halves of their bytes)
                                ws[m][0] = __half2float(ss[m][c * GC + gc]) * 0.0625f;
                                ws[m][1] = __half2float(ss[m][8 * PER + c * GC + gc]) * 0.0625f;
                            }
#pragma unroll
                            for (int j = 0; j < NT; j++) {
                                if (8 * j < rows) {
                                    int d[MT][4];
#pragma unroll
                                    for (int m = 0; m < MT; m++) d[m][0] = d[m][1] = d[m][2] = d[m][3] = Q4_MAGIC;
#pragma unroll
                                    for (int st = 0; st < GS / 32; st++) {
                                        const uint2 b = __ldg(reinterpret_cast<const uint2 *>(xr[j] + grp * GS + 32 * st));
#pragma unroll
                                        for (int m = 0; m < MT; m++) mma_s8(d[m], A[m][st], b.x, b.y);
                                    }
                                    const float *xs = a.xs + (size_t)row0 * G + grp;
                                    const float x0 = __ldg(xs + (size_t)min(8 * j + 2 * t, rows - 1) * G), x1 = __ldg(xs + (size_t)min(8 * j + 2 * t + 1, rows - 1) * G);
#pragma unroll
                                    for (int m = 0; m < MT; m++) {
                                        p[m][j][0] = fmaf(__int_as_float(d[m][0]) - Q4_MAGIC_F, ws[m][0] * x0, p[m][j][0]);
                                        p[m][j][1] = fmaf(__int_as_float(d[m][1]) - Q4_MAGIC_F, ws[m][0] * x1, p[m][j][1]);
                                        p[m][j][2] = fmaf(__int_as_float(d[m][2]) - Q4_MAGIC_F, ws[m][1] * x0, p[m][j][2]);
                                        p[m][j][3] = fmaf(__int_as_float(d[m][3]) - Q4_MAGIC_F, ws[m][1] * x1, p[m][j][3]);
                                    }
                                }
                            }
                        }
                    }
                }
                fetch(4 * (sl + NW) + c, c);
            }
        }
        if (s0 > 0) __syncthreads();  // the last round's partial sums have been read
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int j = 0; j < NT; j++) {
                float *o = red + ((size_t)w * R + 8 * j + 2 * t) * FS + 16 * m + g;
                o[0] = p[m][j][0];
                o[FS] = p[m][j][1];
                o[8] = p[m][j][2];
                o[FS + 8] = p[m][j][3];
            }
        __syncthreads();
        const int nw = min(NW, W.slices - s0);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(tot) / 4); i++) {
            const int e = i * blockDim.x + threadIdx.x;
            if (e < R * FT)
                for (int u = 0; u < nw; u += 2) {
                    const float *o = red + ((size_t)u * R + e / FT) * FS + e % FT;
                    tot[i] += u + 1 < nw ? o[0] + o[R * FS] : o[0];
                }
        }
    }
    if constexpr (!GATED) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(tot) / 4); i++) {
            const int e = i * blockDim.x + threadIdx.x, r = e / FT;
            const int f = blockIdx.x * FT + e % FT;
            if (e < R * FT && r < rows && f < W.n) a.out[(size_t)(row0 + r) * W.n + f] = tot[i];
        }
    } else {
        // the two products of an output are in different threads: through shared memory
        __syncthreads();
#pragma unroll
        for (int i = 0; i < (int)(sizeof(tot) / 4); i++) {
            const int e = i * blockDim.x + threadIdx.x;
            if (e < R * FT) red[(size_t)(e / FT) * FS + e % FT] = tot[i];
        }
        __syncthreads();
        float *h = red + R * FS, *top = h + R * 16;  // [R][16], [R]  (behind the sums: NW >= 2)
        for (int e = threadIdx.x; e < R * 16; e += blockDim.x) {
            const int r = e >> 4, fo = e & 15, f = blockIdx.x * 16 + fo;
            const float v = q4_silu_mul(red[r * FS + fo], red[r * FS + 16 + fo]);
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
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
            for (int e = threadIdx.x; e < R * 16; e += blockDim.x) {
                const int r = e >> 4, fo = e & 15;
                float m = 0.0f;
#pragma unroll
                for (int q = 0; q < CL; q++) {
                    uint32_t at;
                    float v;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(top + r)), "r"(q));
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
                    m = fmaxf(m, v);
                }
                if (r < rows) {
                    const size_t f = (size_t)blockIdx.x * 16 + fo;
                    a.hq[(size_t)(row0 + r) * W.n + f] = wo_quant_level(h[e], m);
                    if (f % GS == 0) a.hs[(size_t)(row0 + r) * (W.n / GS) + f / GS] = m * (1.0f / 127.0f);
                }
            }
            // (no CTA leaves while another may still read its maxima)
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        }
    }
}

template <int GS, int MT, int NT, bool GATED>
cudaError_t launch_q4_rows(const Q4Args &a, cudaStream_t stream) {
    const int NW = a.w.slices >= 8 ? 8 : 4;  // at least four warps own the outputs of the CTA
    const size_t smem = (size_t)NW * 8 * NT * (16 * MT + 4) * sizeof(float);
    auto kern = q4_rows_kernel<GS, MT, NT, GATED>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(GATED ? a.w.tiles : (a.w.tiles + MT - 1) / MT, (a.rows + 8 * NT - 1) / (8 * NT));
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
//   warps 0 .. 7   drain: a thread owns an output (TMEM lane) and RT / 2 rows: p = fma(D, ws xs, p), packed over row pairs; ws in a
//                  register, xs broadcast from shared memory; a slice's p, and the running total, rest in TMEM columns
//   warps 8 .. 11  unpack: 32 bytes of a tile per load, straight from the layout (four chunks ahead in registers), to int8 rows of 128 inputs with
//                  the 128-byte swizzle (K-major A operand); first thread: the rows' levels by TMA (K-major B operand); the xs
//   warp 12        issues the MMAs, two D buffers in turn
// What bounds it is the drain: per D value one conversion, a multiplication for the scales' product and a multiply-add, 128 of either per
// clock and SM at most (64 conversions), against 4,096 or more products per clock in the tensor core.
// With few tiles the inputs are split over the C CTAs of a cluster at multiples of 1,024: every CTA leaves the sums of its pairs of slices
// in its shared memory and each CTA adds up its share of the rows in the one order, reading from the others'.
constexpr int Q4T_THREADS = 416, Q4T_FS = 129;
__host__ __device__ constexpr int q4t_stage(int rt) { return 16384 + rt * 128; }
__host__ __device__ constexpr int q4t_xs(int gs, int rt) { return 2 * (Q4_SLICE / gs) * rt * 4; }
__host__ __device__ constexpr int q4t_sums(int rt) { return rt * Q4T_FS * 4; }  // one pair's sums [RT][129]

__device__ __forceinline__ void ldg_stream8(const void *p, uint32_t *r) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p));
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(const float *p, uint32_t rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// stages: operand stages; np: pairs of slices per CTA (C > 1: also the number of sums kept); grid (C, output tiles, row tiles), cluster (C, P)
template <int GS, int RT, bool GATED>
__global__ void __launch_bounds__(Q4T_THREADS, 1)
    q4_tiles_kernel(const Q4Args a, const __grid_constant__ CUtensorMap xmap, const int stages, const int np, const int C, const int P, int *err) {
    constexpr int GC = Q4_CHUNK / GS, PER = Q4_SLICE / GS, RC = RT / 2, TILES = GATED ? 4 : 8;
    constexpr int HOLD = 2 * RT, TOTAL = 3 * RT, COLS = 4 * RT;  // TMEM: two D buffers, a slice's p, the total
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float *xss = reinterpret_cast<float *>(sm + stages * q4t_stage(RT));  // [2][PER][RT]
    float *sums = xss + q4t_xs(GS, RT) / 4;                              // [C > 1 ? np : 1][RT][129]
    __shared__ __align__(8) uint64_t full[4], empty[4], dfull[2], dempty[2], xfull[2], xempty[2], done;
    __shared__ uint32_t tmem_slot;
    __shared__ float top[RT];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Q4View &W = a.w;
    const int K = W.k, G = K / GS, row0 = blockIdx.z * RT, kc = blockIdx.x;
    const int chunk0 = kc * np * (Q4_PAIR / Q4_CHUNK), chunk1 = min(W.chunks, chunk0 + np * (Q4_PAIR / Q4_CHUNK));
    auto tile_of = [&](int tl) { return min((int)blockIdx.y * TILES + (GATED ? tl & 3 : tl), W.tiles - 1); };

    uint32_t ring[4][2][8];
    const uint8_t *lv[2];
    if (warp >= 8 && warp < 12) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int tl = (warp - 8) + 4 * i;
            const Q4View &M = GATED && tl >= 4 ? a.up : a.w;
            lv[i] = reinterpret_cast<const uint8_t *>(M.levels) + (size_t)tile_of(tl) * W.chunks * 1024 + (lane & 15) * 64 + (lane >> 4) * 32;
        }
        // (the weights are written once, when the matrix is made: their loads need not wait for the kernel before this one)
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (chunk0 + c < chunk1) ldg_stream8(lv[i] + (size_t)(chunk0 + c) * 1024, ring[c][i]);
    }
    pdl_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < 4; i++) mbar_init(full + i, 129), mbar_init(empty + i, 1);
        for (int i = 0; i < 2; i++) mbar_init(dfull + i, 1), mbar_init(dempty + i, 8), mbar_init(xfull + i, 128), mbar_init(xempty + i, 8);
        mbar_init(&done, 1);
        mbar_fence_init();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = tmem_slot;
    pdl_wait();

    if (warp < 8) {
        // ---- drain
        const int quad = warp & 3, col0 = (warp >> 2) * RC, tl = 2 * quad + (lane >> 4);
        const uint32_t mine = tbase + ((uint32_t)(quad * 32) << 16) + col0;
        const Q4View &M = GATED && tl >= 4 ? a.up : a.w;
        const __half *sc = M.scales + ((size_t)tile_of(tl) * W.slices * Q4_TILE + (lane & 15)) * PER;
        float2 p[RC / 2];
        bool ok = true;
        int gi = 0;  // groups drained
        __align__(16) __half wsn[PER], wsc[PER];
        auto fetch_ws = [&](int sl) {
            const __half *s = sc + (size_t)sl * Q4_TILE * PER;
            if constexpr (PER == 4) *reinterpret_cast<uint2 *>(wsn) = __ldg(reinterpret_cast<const uint2 *>(s));
            else
#pragma unroll
                for (int i = 0; i < PER / 8; i++) reinterpret_cast<uint4 *>(wsn)[i] = __ldg(reinterpret_cast<const uint4 *>(s) + i);
        };
        const int sl0 = chunk0 / 4, sl1 = (chunk1 + 3) / 4;
        fetch_ws(sl0);
        for (int sl = sl0; sl < sl1 && ok; sl++) {
            const int slot = (sl - sl0) & 1;
#pragma unroll
            for (int i = 0; i < PER; i++) wsc[i] = wsn[i];
            if (sl + 1 < sl1) fetch_ws(sl + 1);
#pragma unroll
            for (int i = 0; i < RC / 2; i++) p[i] = make_float2(0.0f, 0.0f);
            ok = mbar_wait_bounded_quiet(xfull + slot, (uint32_t)((sl - sl0) >> 1) & 1u, err, 81);
            const float *xsl = xss + slot * PER * RT + col0;
#pragma unroll
            for (int g = 0; g < PER; g++) {
                if (4 * sl + g / GC < chunk1 && ok) {
                    const int buf = gi & 1;
                    ok = mbar_wait_bounded_quiet(dfull + buf, (uint32_t)(gi >> 1) & 1u, err, 82);
                    ok = __all_sync(0xffffffffu, ok);
                    tc_fence_after();
                    const float w = __half2float(wsc[g]) * 0.0625f;  // (1 / 16: the levels are in the upper halves of their bytes)
                    const float2 w2 = make_float2(w, w);
                    constexpr int B = RC < 32 ? RC : 32;  // columns read at a time
#pragma unroll
                    for (int c = 0; c < RC; c += B) {
                        uint32_t r[B];
                        if constexpr (B == 16) tmem_ld16(mine + buf * RT, r);
                        else tmem_ld32(mine + buf * RT + c, r);
                        tmem_wait_ld();
                        if (c + B == RC) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(dempty + buf);
                        }
#pragma unroll
                        for (int j = 0; j < B; j += 4) {
                            const float4 x = *reinterpret_cast<const float4 *>(xsl + g * RT + c + j);
                            float2 &p0 = p[(c + j) / 2], &p1 = p[(c + j) / 2 + 1];
                            p0 = __ffma2_rn(make_float2((float)(int)r[j], (float)(int)r[j + 1]), __fmul2_rn(w2, make_float2(x.x, x.y)), p0);
                            p1 = __ffma2_rn(make_float2((float)(int)r[j + 2], (float)(int)r[j + 3]), __fmul2_rn(w2, make_float2(x.z, x.w)), p1);
                        }
                    }
                    gi++;
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(xempty + slot);
            // the end of the slice: hold p, or add it to the slice before and the pair to the total
            if (!(sl & 1) && sl + 1 < sl1) {
                if constexpr (RC == 16) tmem_st16(mine + HOLD, reinterpret_cast<uint32_t *>(p));
                else
#pragma unroll
                    for (int i = 0; i < RC / 32; i++) tmem_st32(mine + HOLD + 32 * i, reinterpret_cast<uint32_t *>(p) + 32 * i);
                tmem_wait_st();
            } else {
                const int pair = (sl - sl0) >> 1;
#pragma unroll
                for (int i = 0; i < RC / 16; i++) {
                    uint32_t r[16];
                    if (sl & 1) {
                        tmem_ld16(mine + HOLD + 16 * i, r);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            p[8 * i + j] = __fadd2_rn(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), p[8 * i + j]);
                    }
                    if (C == 1) {
                        if (pair > 0) {
                            tmem_ld16(mine + TOTAL + 16 * i, r);
                            tmem_wait_ld();
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; j++) r[j] = 0u;
                        }
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            p[8 * i + j] = __fadd2_rn(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), p[8 * i + j]);
                        if (sl + 1 < sl1) {
                            tmem_st16(mine + TOTAL + 16 * i, reinterpret_cast<uint32_t *>(p + 8 * i));
                            tmem_wait_st();
                        }
                    }
                }
                if (C > 1 || sl + 1 == sl1) {
                    float *o = sums + ((size_t)(C > 1 ? pair : 0) * RT + col0) * Q4T_FS + quad * 32 + lane;
#pragma unroll
                    for (int j = 0; j < RC / 2; j++) {
                        o[2 * j * Q4T_FS] = p[j].x;
                        o[(2 * j + 1) * Q4T_FS] = p[j].y;
                    }
                }
            }
        }
    } else if (warp < 12) {
        // ---- unpack
        const int u = tid - 256, f = lane & 15, h = lane >> 4, row = row0 + u;
        bool ok = true;
        float xn[PER];
        auto fetch_xs = [&](int sl) {
#pragma unroll
            for (int i = 0; i < PER; i++) xn[i] = u < RT && row < a.rows && sl * PER + i < G ? __ldg(a.xs + (size_t)row * G + sl * PER + i) : 0.0f;
        };
        fetch_xs(chunk0 / 4);
        int st = 0;
        uint32_t ph = 0;  // the phase of the stages' empty barriers that the next round waits for
        for (int base = chunk0; base < chunk1 && ok; base += 4) {
            const int sl = base / 4, n = sl - chunk0 / 4;
            if (n >= 2) ok = mbar_wait_bounded_quiet(xempty + (n & 1), (uint32_t)((n >> 1) - 1) & 1u, err, 83);
            if (u < RT)
#pragma unroll
                for (int i = 0; i < PER; i++) xss[((n & 1) * PER + i) * RT + u] = xn[i];
            mbar_arrive(xfull + (n & 1));
            if (base + 4 < chunk1) fetch_xs(sl + 1);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int chunk = base + c;
                if (chunk < chunk1 && ok) {
                    uint8_t *A = sm + st * q4t_stage(RT);
                    if (chunk - chunk0 >= stages) ok = mbar_wait_bounded_quiet(empty + st, ph ^ 1u, err, 84);
                    if (u == 0) {
                        mbar_expect_tx(full + st, RT * 128);
                        tma_load_2d(A + 16384, &xmap, chunk * Q4_CHUNK, row0, full + st);
                    }
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        uint8_t *o = A + ((warp - 8) + 4 * i) * 2048 + f * 128;
#pragma unroll
                        for (int s = 0; s < 4; s++) {
                            const uint32_t w0 = ring[c][i][s], w1 = ring[c][i][4 + s];
                            *reinterpret_cast<uint4 *>(o + (((2 * s + h) ^ (f & 7)) << 4)) =
                                make_uint4((w0 << 4) & 0xF0F0F0F0u, w0 & 0xF0F0F0F0u, (w1 << 4) & 0xF0F0F0F0u, w1 & 0xF0F0F0F0u);
                        }
                        if (chunk + 4 < chunk1) ldg_stream8(lv[i] + (size_t)(chunk + 4) * 1024, ring[c][i]);
                    }
                    fence_proxy_async();
                    mbar_arrive(full + st);
                    if (++st == stages) st = 0, ph ^= 1u;
                }
            }
        }
        if (u == 0 && *reinterpret_cast<volatile int *>(err) != 0)  // a wait ran out: the copies in flight get a bounded time to land
            for (int i = 0; i < stages; i++) mbar_drain(full + i, ph);
    } else if (elect_one()) {
        // ---- MMA issue
        constexpr uint32_t idesc = umma_idesc_i8(128, RT, 0, 0, 1, 1);
        const uint32_t sbase = smem_u32(sm);
        int st = 0, gi = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int chunk = chunk0; chunk < chunk1 && ok; chunk++) {
            ok = mbar_wait_bounded_quiet(full + st, ph, err, 85);
            tc_fence_after();
            const uint32_t A = sbase + st * q4t_stage(RT), B = A + 16384;
#pragma unroll
            for (int gc = 0; gc < GC; gc++) {
                const int buf = gi & 1;
                if (gi >= 2 && ok) ok = mbar_wait_bounded_quiet(dempty + buf, (uint32_t)((gi >> 1) - 1) & 1u, err, 86);
                if (ok) {
                    tc_fence_after();
#pragma unroll
                    for (int s = 0; s < GS / 32; s++) {
                        const int at = gc * GS + 32 * s;
                        umma_i8(tbase + buf * RT, umma_desc(A + at, 16, 1024, 2), umma_desc(B + at, 16, 1024, 2), idesc, s > 0);
                    }
                    umma_commit(dfull + buf);
                }
                gi++;
            }
            umma_commit(empty + st);
            if (++st == stages) st = 0, ph ^= 1u;
        }
        umma_commit(&done);
        mbar_drain(&done, 0);  // (no MMA and no arrival of one is in flight when the CTA ends)
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(COLS));
    if (C > 1) cluster_sync_all();  // (the clusters of 128-wide groups and C = 1 have nothing to read here yet)

    // ---- the totals of this CTA's share of the rows, a warp per row, lanes along the outputs
    const int share = (RT + C - 1) / C, r0 = kc * share, r1 = min(min(r0 + share, RT), a.rows - row0);
    const int pairs = (W.chunks + 7) / 8;
    const uint32_t prank = (uint32_t)(blockIdx.y % P) * C;
    auto total = [&](int r, int f) {
        if (C == 1) return sums[r * Q4T_FS + f];
        float t = 0.0f;
        for (int q = 0; q < pairs; q++) t += ld_cluster(sums + ((size_t)(q % np) * RT + r) * Q4T_FS + f, prank + q / np);
        return t;
    };
    if constexpr (!GATED) {
        for (int r = r0 + warp; r < r1; r += Q4T_THREADS / 32)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int f = blockIdx.y * 128 + 32 * i + lane;
                const float v = total(r, 32 * i + lane);
                if (f < W.n) a.out[(size_t)(row0 + r) * W.n + f] = v;
            }
    } else {
        for (int pass = a.hq && GS == 128 ? 0 : 1; pass < 2; pass++) {
            if (pass == 1 && a.hq && GS == 128) cluster_sync_all();  // the two CTAs of a group's halves have their maxima
            for (int r = r0 + warp; r < r1; r += Q4T_THREADS / 32) {
                float v[2];
                uint32_t m[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    v[i] = q4_silu_mul(total(r, 32 * i + lane), total(r, 64 + 32 * i + lane));
                    m[i] = a.hq ? __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fabsf(v[i]), 0.0f))) : 0u;  // (a NaN counts as 0)
                }
                if (GS >= 64) m[0] = m[1] = max(m[0], m[1]);
                if (pass == 0) {
                    if (lane == 0) top[r] = __uint_as_float(m[0]);
                    continue;
                }
                if (a.hq && GS == 128) {
                    const uint32_t other = (uint32_t)(blockIdx.y % P ^ 1) * C + kc;
                    m[0] = m[1] = max(m[0], __float_as_uint(ld_cluster(top + r, other)));
                }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int f = blockIdx.y * 64 + 32 * i + lane;
                    const size_t at = (size_t)(row0 + r) * W.n + f;
                    if (f < W.n) {
                        if (a.out) a.out[at] = v[i];
                        if (a.hq) {
                            a.hq[at] = wo_quant_level(v[i], __uint_as_float(m[i]));
                            if (f % GS == 0) a.hs[at / GS] = __uint_as_float(m[i]) * (1.0f / 127.0f);
                        }
                    }
                }
            }
        }
    }
    if (C > 1 || P > 1) cluster_sync_all();  // no CTA leaves while another may still read its sums or maxima
}

template <int GS, int RT, bool GATED>
cudaError_t launch_q4_tiles(const Q4Args &a, int C, Q4EncodeFn enc, int *err, cudaStream_t stream) {
    const int pairs = (a.w.slices + 1) / 2, np = (pairs + C - 1) / C;
    C = (pairs + np - 1) / np;
    const int P = GATED && a.hq && GS == 128 ? 2 : 1;
    const int fixed = 1024 + q4t_xs(GS, RT) + q4t_sums(RT) * (C > 1 ? np : 1), most = 226 * 1024;
    int stages = (most - fixed) / q4t_stage(RT);
    if (stages < 2) return cudaErrorInvalidValue;
    if (stages > 4) stages = 4;
    const int smem = fixed + stages * q4t_stage(RT);
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)a.w.k, (cuuint64_t)a.rows}, strides[1] = {(cuuint64_t)a.w.k};
    const cuuint32_t box[2] = {Q4_CHUNK, RT}, es[2] = {1, 1};
    if (!enc || enc(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(a.xq), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    auto kern = q4_tiles_kernel<GS, RT, GATED>;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    const int tiles = GATED ? 4 : 8;
    cfg.gridDim = dim3(C, (a.w.tiles + tiles - 1) / tiles, (a.rows + RT - 1) / RT);
    cfg.blockDim = dim3(Q4T_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = C;
    at[1].val.clusterDim.y = P;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = C * P > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, a, map, stages, np, C, P, err);
}

// Which rows per tile and how many CTAs along the inputs: the least estimated time, in clocks.  A group costs a CTA its drain (measured:
// q4t_group) and a CTA costs its start and end; CTAs run one per SM, in waves.
struct Q4Plan {
    int rt, c;
};
inline Q4Plan q4_plan(const Q4Args &a, bool gated, int n_sm) {
    const int pairs = (a.w.slices + 1) / 2, tiles = (a.w.tiles + (gated ? 3 : 7)) / (gated ? 4 : 8), P = gated && a.hq && a.w.gs == 128 ? 2 : 1;
    Q4Plan best = {128, 1};
    double least = 1e300;
    for (int rt = 32; rt <= 128; rt *= 2) {
        const double group = rt == 128 ? 330.0 : rt == 64 ? 180.0 : 120.0;
        for (int c = 1; c * P <= 8 && c <= pairs; c++) {
            const int np = (pairs + c - 1) / c;
            if ((pairs + np - 1) / np != c) continue;
            if (1024 + q4t_xs(a.w.gs, rt) + q4t_sums(rt) * (c > 1 ? np : 1) + 2 * q4t_stage(rt) > 226 * 1024) continue;
            const long long ctas = (long long)c * tiles * ((a.rows + rt - 1) / rt), slots = n_sm / (c * P) * (c * P);
            const double time = (double)((ctas + slots - 1) / slots) * (3000.0 + (c > 1 ? 1500.0 : 0.0) + (double)np * (Q4_PAIR / a.w.gs) * group);
            if (time < least) least = time, best = {rt, c};
        }
    }
    return best;
}

template <int GS>
cudaError_t launch_q4_gs(const Q4Args &a, bool gated, int n_sm, Q4EncodeFn enc, int *err, cudaStream_t stream) {
#define Q4_BY_ROWS(MT_, GATED_)                                           \
    if (a.rows <= 8) return launch_q4_rows<GS, MT_, 1, GATED_>(a, stream); \
    if (a.rows <= 16) return launch_q4_rows<GS, MT_, 2, GATED_>(a, stream); \
    const Q4Plan plan = q4_plan(a, GATED_, n_sm);                          \
    if (plan.rt == 32) return launch_q4_tiles<GS, 32, GATED_>(a, plan.c, enc, err, stream); \
    if (plan.rt == 64) return launch_q4_tiles<GS, 64, GATED_>(a, plan.c, enc, err, stream); \
    return launch_q4_tiles<GS, 128, GATED_>(a, plan.c, enc, err, stream)
    if (gated) { Q4_BY_ROWS(2, true); }
    Q4_BY_ROWS(1, false);
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
