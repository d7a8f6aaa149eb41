// Products of 8-bit rows with 4-bit weight matrices, and the gated feed-forward product built on them.
//
//   y[r][f] = sum over groups of GS inputs  xs[r][g] ws[f][g] D,   D = sum over the group of xq[r][k] wq[f][k]   (an exact integer)
//
// xq, xs: the rows as the quantisers of this library leave them (int8 levels, one fp32 scale per group); wq: levels -8 .. 7, ws: f16.
// The sum over groups has one order, whatever kernel runs and however many rows a pass has: inputs are cut into slices of 512, a
// slice's groups are a chain p = fma(D, ws xs, p) in ascending order from 0, and the slices are added in ascending order from 0.
// So a row's result does not depend on the other rows of the pass.
#pragma once
#include "attn_decode.cuh"

namespace rq {

constexpr int Q4_TILE = 16;    // outputs per tile of the layout
constexpr int Q4_CHUNK = 128;  // inputs per chunk: a (tile, chunk) is 1 KB
constexpr int Q4_SLICE = 512;  // inputs per slice of the sum's order

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

struct Q4Args {
    Q4View w, up;        // the matrix; the gated product's second matrix
    const int8_t *xq;    // [rows][k]
    const float *xs;     // [rows][k / gs]
    int rows;
    float *out;          // [rows][n], or null (gated product)
    int8_t *hq;          // [rows][n] and [rows][n / gs]: the gated product's rows in 8 bits, or null
    float *hs;
};

// mm: out = x W^T;  gated: out = silu(x W^T) (x Up^T)
cudaError_t launch_q4(const Q4Args &a, bool gated, cudaStream_t stream);
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
                for (int u = 0; u < nw; u++) tot[i] += red[((size_t)u * R + e / FT) * FS + e % FT];
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

template <int GS>
cudaError_t launch_q4_gs(const Q4Args &a, bool gated, cudaStream_t stream) {
#define Q4_BY_ROWS(MT_, GATED_)                                           \
    if (a.rows <= 8) return launch_q4_rows<GS, MT_, 1, GATED_>(a, stream); \
    if (a.rows <= 16) return launch_q4_rows<GS, MT_, 2, GATED_>(a, stream); \
    if (a.rows <= 32) return launch_q4_rows<GS, MT_, 4, GATED_>(a, stream); \
    return launch_q4_rows<GS, MT_, 8, GATED_>(a, stream)
    if (gated) { Q4_BY_ROWS(2, true); }
    Q4_BY_ROWS(1, false);
#undef Q4_BY_ROWS
}

cudaError_t launch_q4(const Q4Args &a, bool gated, cudaStream_t stream) {
    switch (a.w.gs) {
        case 32: return launch_q4_gs<32>(a, gated, stream);
        case 64: return launch_q4_gs<64>(a, gated, stream);
        default: return launch_q4_gs<128>(a, gated, stream);
    }
}

#endif  // RQ_Q4_INSTANTIATE

}  // namespace rq
