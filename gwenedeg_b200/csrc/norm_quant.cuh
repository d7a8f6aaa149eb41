// The step between two sublayers of a forward pass: the residual addition, the RMS norm and the 8-bit rows that the next matrix
// product reads (the reference's rmsnorm, src/forward.c:886, followed by its quantize, :803), in one pass over the rows.
#pragma once
#include "attn_decode.cuh"

namespace rq {

// Per row:  x' = x + d (each sum rounded once; d null: x' = x);  inv = 1 / sqrt(mean(x'^2) + eps);  v = x' w;  per group of GS
// values  m = max |v|,  level = the framework's quantiser on (v, m),  scale = m (1 / 127) inv;  optionally y = v inv.
// inv is a factor of every v of the row, so it cancels out of level = 127 v / m and goes into the scale alone: the levels are
// decided by x' and w only (element by element, correctly rounded operations) and do not depend on the order of the row's sum.
//
// One CTA per row, thread t holds the float4s t, t + T, ... of the row in registers (V of them): x and d are read once, x', the
// levels, the scales and y written once.  T and V depend on the row's width only, so a row's sum has one order whatever the
// number of rows.  A group is 8, 16 or 32 adjacent lanes.  Sums in fp32: per thread, then a warp tree, then the warps in order.
// Bound by the rows' bytes: 2048 x 4096 (x, d read, x', levels written) 19.0 us = 5.8 TB/s, 4096 x 8192 70 us = 6.2 TB/s; a single row
// of 4096 takes 2.4 us, the latency of a launch, one load and two reductions.
struct NormQuantArgs {
    const float *x, *delta, *w;
    float *x_out, *y;
    int8_t *xq;
    float *xs;
    int dim;
    float eps;
};

template <int GS, int V>
__global__ void __launch_bounds__(1024) add_norm_quant_kernel(const NormQuantArgs a) {
    const int tid = threadIdx.x, T = blockDim.x, n4 = a.dim / 4;
    const size_t row = blockIdx.x;
    __shared__ float red[32];
    pdl_launch_dependents();
    pdl_wait();
    const float4 *x = reinterpret_cast<const float4 *>(a.x + row * a.dim);
    float4 v[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        const int i = j * T + tid;
        v[j] = i < n4 ? x[i] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (a.delta) {
        const float4 *d = reinterpret_cast<const float4 *>(a.delta + row * a.dim);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int i = j * T + tid;
            if (i < n4) {
                const float4 e = d[i];
                v[j].x += e.x, v[j].y += e.y, v[j].z += e.z, v[j].w += e.w;
            }
        }
    }
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < V; j++) {
        const int i = j * T + tid;
        if (a.x_out && i < n4) reinterpret_cast<float4 *>(a.x_out + row * a.dim)[i] = v[j];
        ss = fmaf(v[j].x, v[j].x, ss);
        ss = fmaf(v[j].y, v[j].y, ss);
        ss = fmaf(v[j].z, v[j].z, ss);
        ss = fmaf(v[j].w, v[j].w, ss);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if ((tid & 31) == 0) red[tid >> 5] = ss;
    __syncthreads();
    ss = 0.0f;
    for (int i = 0; i < T / 32; i++) ss += red[i];
    const float inv = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
#pragma unroll
    for (int j = 0; j < V; j++) {
        const int i = j * T + tid;
        float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < n4) {
            const float4 w = reinterpret_cast<const float4 *>(a.w)[i];
            u = make_float4(v[j].x * w.x, v[j].y * w.y, v[j].z * w.z, v[j].w * w.w);
        }
        if (a.xq) {
            float m = fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(u.z), fabsf(u.w)));
#pragma unroll
            for (int o = GS / 8; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (i < n4) {
                const float t = quant_top(m);
                char4 q;
                q.x = wo_quant_level(u.x, t), q.y = wo_quant_level(u.y, t), q.z = wo_quant_level(u.z, t), q.w = wo_quant_level(u.w, t);
                reinterpret_cast<char4 *>(a.xq + row * a.dim)[i] = q;
                if (i % (GS / 4) == 0) a.xs[row * (a.dim / GS) + i / (GS / 4)] = quant_scale(m) * inv;
            }
        }
        if (a.y && i < n4) reinterpret_cast<float4 *>(a.y + row * a.dim)[i] = make_float4(u.x * inv, u.y * inv, u.z * inv, u.w * inv);
    }
}

constexpr int NORM_MAX_DIM = 32768;  // 1024 threads of 8 float4s

inline cudaError_t launch_add_norm_quant(const NormQuantArgs &a, int rows, int gs, cudaStream_t stream) {
    const int n4 = a.dim / 4;
    int T = ((n4 + 1) / 2 + 31) / 32 * 32;
    T = T < 64 ? 64 : T > 1024 ? 1024 : T;
    const int V = (n4 + T - 1) / T;
#define NQ(GS_, V_) return launch_pdl(add_norm_quant_kernel<GS_, V_>, dim3(rows), dim3(T), 0, stream, a)
#define NQV(GS_)          \
    if (V <= 2) NQ(GS_, 2); \
    if (V <= 4) NQ(GS_, 4); \
    NQ(GS_, 8)
    if (gs == 32) { NQV(32); }
    if (gs == 64) { NQV(64); }
    NQV(128);
#undef NQV
#undef NQ
}

}  // namespace rq
