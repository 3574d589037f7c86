// qk_rope.hip -- RMS norm of each head's query and key and the position
// rotation in one pass, and its backward.
//
//   u = x r, r = (mean x^2 + eps)^(-1/2), z = u w      (norm; else z = x)
//   y_a = z_a cos - z_b sin,  y_b = z_b cos + z_a sin   for each rotated pair (a, b)
// Pair i is (i, i + rot/2), or (2i, 2i + 1) interleaved; its angle is a row
// of the table chosen by the token's position on the pair's axis.  Backward,
// for g = dL/dy:
//   dz = the rotation by the opposite angle of g
//   dw = sum over tokens and heads of dz u,   du = dz w
//   dx = r (du - u mean(du u))
//
// A lane holds 8 values of a head: both halves of 4 pairs (two 4-value loads
// rot/2 apart, or 8 neighbours interleaved), or 8 values behind the rotated
// part, so no value crosses lanes but in the norm's sums.  The dim / 8 lanes
// of a token keep its cosines and sines in registers and walk over heads.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qk_rope.hpp"
#include "vec_io.hpp"

namespace coset {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxGroups = 512;   // backward: workgroups along the tokens, one row of weight sums each

struct Lane {
    int first, second;   // element of x[0..3] and of x[4..7]
    bool turned;
    bool on;
};

// With pairs rot/2 apart, lane l < rot/8 holds pairs 4l..4l+3; else lane l holds
// elements 8l..8l+7.
__device__ __forceinline__ Lane lane_of(const RopeArgs& a, int l)
{
    Lane r;
    r.on = 8 * l < a.dim;
    r.turned = 8 * l < a.rot;
    const bool apart = r.turned && !a.interleaved;
    r.first = apart ? 4 * l : 8 * l;
    r.second = apart ? a.rot / 2 + 4 * l : 8 * l + 4;
    return r;
}

template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t at, const Lane& l, bool vec, float (&x)[8])
{
    load_n<DT, 4>(p, at + l.first, vec, x);
    load_n<DT, 4>(p, at + l.second, vec, x + 4);
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t at, const Lane& l, const float (&x)[8])
{
    store_n<DT, 4>(p, at + l.first, x);
    store_n<DT, 4>(p, at + l.second, x + 4);
}

__device__ __forceinline__ void load_weight(const void* w, int dt, const Lane& l, float (&x)[8])
{
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 1.f;
    if (!w || !l.on) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int e = j < 4 ? l.first + j : l.second + j - 4;
        x[j] = dt == DT_F32 ? load1<DT_F32>(w, e) : dt == DT_BF16 ? load1<DT_BF16>(w, e) : load1<DT_F16>(w, e);
    }
}

// cosines and sines of the lane's four pairs 4l..4l+3
__device__ __forceinline__ void load_turn(const RopeArgs& a, int l, int64_t t, const Lane& ln, float (&c)[4], float (&s)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[i] = 1.f;
        s[i] = 0.f;
    }
    if (!ln.turned) return;
    const int half = a.rot / 2;
    if (a.axes == 1) {
        const int64_t p = min(max(a.pos[t], (int64_t)0), a.length - 1);
        const float4 cc = *reinterpret_cast<const float4*>(a.table + p * a.rot + 4 * l);
        const float4 ss = *reinterpret_cast<const float4*>(a.table + p * a.rot + half + 4 * l);
        c[0] = cc.x;
        c[1] = cc.y;
        c[2] = cc.z;
        c[3] = cc.w;
        s[0] = ss.x;
        s[1] = ss.y;
        s[2] = ss.z;
        s[3] = ss.w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int pair = 4 * l + i;
        int axis = 0;
        for (int k = 0; k + 1 < a.axes; ++k) axis += pair >= a.bound[k] ? 1 : 0;
        const int64_t p = min(max(a.pos[axis * a.pos_axis + t], (int64_t)0), a.length - 1);
        c[i] = a.table[p * a.rot + pair];
        s[i] = a.table[p * a.rot + half + pair];
    }
}

// (x_a, x_b) turned by +-angle; pairs (x[i], x[4+i]) or (x[2i], x[2i+1])
__device__ __forceinline__ void turn(float (&x)[8], const float (&c)[4], const float (&s)[4], bool near, float sign)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float u = near ? x[2 * i] : x[i], v = near ? x[2 * i + 1] : x[4 + i];
        const float si = sign * s[i];
        const float y = u * c[i] - v * si, z = v * c[i] + u * si;
        if (near) {
            x[2 * i] = y;
            x[2 * i + 1] = z;
        } else {
            x[i] = y;
            x[4 + i] = z;
        }
    }
}

template <int GW>
__device__ __forceinline__ float group_sum(float v)
{
#pragma unroll
    for (int o = 1; o < GW; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Heads [h0, h1) of the queries followed by the keys.
template <int DT, int GW, bool NEAR>
__global__ void __launch_bounds__(kThreads) rope_fwd_kernel(RopeArgs a, int per)
{
    const int l = threadIdx.x % GW;
    const int64_t t = (int64_t)blockIdx.x * (kThreads / GW) + threadIdx.x / GW;
    if (t >= a.n) return;
    const Lane ln = lane_of(a, l);
    float c[4], s[4], wq[8], wk[8];
    load_turn(a, l, t, ln, c, s);
    load_weight(a.q.w, a.w_dtype, ln, wq);
    load_weight(a.k.w, a.w_dtype, ln, wk);
    const int h0 = blockIdx.y * per, h1 = min(h0 + per, a.q.heads + a.k.heads);
    const float mean = 1.f / (float)a.dim;
    for (int h = h0; h < h1; ++h) {
        const bool key = h >= a.q.heads;
        const RopeSide& sd = key ? a.k : a.q;
        const int hh = key ? h - a.q.heads : h;
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (ln.on) load8<DT>(sd.x, t * sd.x_tok + hh * sd.x_head, ln, sd.vec, x);
        if (a.norm) {
            float sq = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) sq = fmaf(x[j], x[j], sq);
            const float r = 1.f / sqrtf(fmaf(group_sum<GW>(sq), mean, a.eps));
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = x[j] * r * (key ? wk[j] : wq[j]);
        }
        turn(x, c, s, NEAR, 1.f);
        if (ln.on) store8<DT>(sd.out, (t * sd.heads + hh) * (int64_t)a.dim, ln, x);
    }
}

template <int DT, int GW, bool NEAR>
__global__ void __launch_bounds__(kThreads) rope_bwd_kernel(RopeArgs a)
{
    constexpr int kTokens = kThreads / GW;
    const int l = threadIdx.x % GW;
    const Lane ln = lane_of(a, l);
    float wq[8], wk[8], dq[8], dk[8];
    load_weight(a.q.w, a.w_dtype, ln, wq);
    load_weight(a.k.w, a.w_dtype, ln, wk);
#pragma unroll
    for (int j = 0; j < 8; ++j) dq[j] = dk[j] = 0.f;
    const float mean = 1.f / (float)a.dim;
    for (int64_t t = (int64_t)blockIdx.x * kTokens + threadIdx.x / GW; t < a.n; t += (int64_t)gridDim.x * kTokens) {
        float c[4], s[4];
        load_turn(a, l, t, ln, c, s);
        for (int h = 0; h < a.q.heads + a.k.heads; ++h) {
            const bool key = h >= a.q.heads;
            const RopeSide& sd = key ? a.k : a.q;
            const int hh = key ? h - a.q.heads : h;
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, g[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (ln.on) {
                load8<DT>(sd.g, t * sd.g_tok + hh * sd.g_head, ln, sd.vec, g);
                if (a.norm) load8<DT>(sd.x, t * sd.x_tok + hh * sd.x_head, ln, sd.vec, x);
            }
            turn(g, c, s, NEAR, -1.f);
            if (a.norm) {
                float sq = 0.f, du[8], dot = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    sq = fmaf(x[j], x[j], sq);
                    du[j] = g[j] * (key ? wk[j] : wq[j]);
                    dot = fmaf(du[j], x[j], dot);
                }
                const float r = 1.f / sqrtf(fmaf(group_sum<GW>(sq), mean, a.eps));
                const float m = group_sum<GW>(dot) * r * mean;   // mean(du u)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float u = x[j] * r;
                    const float add = g[j] * u;
                    if (key)
                        dk[j] += add;
                    else
                        dq[j] += add;
                    g[j] = r * fmaf(-u, m, du[j]);
                }
            }
            if (ln.on) store8<DT>(sd.out, (t * sd.heads + hh) * (int64_t)a.dim, ln, g);
        }
    }
    if (!a.partial) return;
    // the workgroup's tokens in a fixed order
    __shared__ float sh[2][kTokens][GW * 8];
    const int row = threadIdx.x / GW;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        sh[0][row][j * GW + l] = dq[j];
        sh[1][row][j * GW + l] = dk[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * GW * 8; i += kThreads) {
        const int side = i / (GW * 8), e = i % (GW * 8);
        float v = 0.f;
        for (int r = 0; r < kTokens; ++r) v += sh[side][r][e];
        const Lane le = lane_of(a, e % GW);
        const int j = e / GW;
        if (le.on) a.partial[((int64_t)blockIdx.x * 2 + side) * a.dim + (j < 4 ? le.first + j : le.second + j - 4)] = v;
    }
}

__device__ __forceinline__ void store_any(void* p, int dt, int64_t i, float v)
{
    if (dt == DT_F32)
        store1<DT_F32>(p, i, v);
    else if (dt == DT_BF16)
        store1<DT_BF16>(p, i, v);
    else
        store1<DT_F16>(p, i, v);
}

// The weights' gradients: 16 columns a workgroup, 16 threads of partials
// each, summed in a fixed order.
__global__ void __launch_bounds__(kThreads) rope_weight_kernel(RopeArgs a, int groups)
{
    __shared__ float sh[16][17];
    const int col = threadIdx.x % 16, part = threadIdx.x / 16;
    const int e = blockIdx.x * 16 + col;
    const int side = blockIdx.y;
    float v = 0.f;
    if (e < a.dim)
        for (int g = part; g < groups; g += 16) v += a.partial[((int64_t)g * 2 + side) * a.dim + e];
    sh[part][col] = v;
    __syncthreads();
    if (part == 0 && e < a.dim) {
        float t = 0.f;
        for (int p = 0; p < 16; ++p) t += sh[p][col];
        void* out = side ? a.gw_k : a.gw_q;   // either may be unwanted
        if (out) store_any(out, a.w_dtype, e, t);
    }
}

template <int DT, int GW, bool NEAR>
hipError_t launch_fwd(const RopeArgs& a, hipStream_t s)
{
    const int heads = a.q.heads + a.k.heads;
    const int64_t rows = (a.n + kThreads / GW - 1) / (kThreads / GW);
    // one head a lane group until the grid holds 8 workgroups per CU
    int per = 1;
    while (per < heads && rows * ((heads + 2 * per - 1) / (2 * per)) >= 2048) per *= 2;
    hipLaunchKernelGGL((rope_fwd_kernel<DT, GW, NEAR>), dim3((unsigned)rows, (heads + per - 1) / per), dim3(kThreads), 0,
                       s, a, per);
    return hipGetLastError();
}

template <int DT, int GW, bool NEAR>
hipError_t launch_bwd(const RopeArgs& a, hipStream_t s)
{
    const int groups = rope_bwd_groups(a.n, a.dim);
    hipError_t e = hipSuccess;
    if (groups > 0) {
        hipLaunchKernelGGL((rope_bwd_kernel<DT, GW, NEAR>), dim3(groups), dim3(kThreads), 0, s, a);
        e = hipGetLastError();
    }
    if (e != hipSuccess || (!a.gw_q && !a.gw_k)) return e;
    hipLaunchKernelGGL(rope_weight_kernel, dim3((a.dim + 15) / 16, 2), dim3(kThreads), 0, s, a, groups);
    return hipGetLastError();
}

int lanes_of(int dim)
{
    int g = 4;
    while (8 * g < dim) g *= 2;
    return g;
}

template <int DT, bool NEAR, bool BWD>
hipError_t by_width(const RopeArgs& a, hipStream_t s)
{
    switch (lanes_of(a.dim)) {
    case 4: return BWD ? launch_bwd<DT, 4, NEAR>(a, s) : launch_fwd<DT, 4, NEAR>(a, s);
    case 8: return BWD ? launch_bwd<DT, 8, NEAR>(a, s) : launch_fwd<DT, 8, NEAR>(a, s);
    case 16: return BWD ? launch_bwd<DT, 16, NEAR>(a, s) : launch_fwd<DT, 16, NEAR>(a, s);
    case 32: return BWD ? launch_bwd<DT, 32, NEAR>(a, s) : launch_fwd<DT, 32, NEAR>(a, s);
    default: return BWD ? launch_bwd<DT, 64, NEAR>(a, s) : launch_fwd<DT, 64, NEAR>(a, s);
    }
}

template <bool BWD>
hipError_t by_type(const RopeArgs& a, hipStream_t s)
{
    switch (a.dtype) {
    case DT_F32: return a.interleaved ? by_width<DT_F32, true, BWD>(a, s) : by_width<DT_F32, false, BWD>(a, s);
    case DT_BF16: return a.interleaved ? by_width<DT_BF16, true, BWD>(a, s) : by_width<DT_BF16, false, BWD>(a, s);
    default: return a.interleaved ? by_width<DT_F16, true, BWD>(a, s) : by_width<DT_F16, false, BWD>(a, s);
    }
}

}  // namespace

int rope_bwd_groups(int64_t n, int dim)
{
    const int64_t rows = (n + kThreads / lanes_of(dim) - 1) / (kThreads / lanes_of(dim));
    return (int)(rows < kMaxGroups ? rows : kMaxGroups);
}

hipError_t launch_rope_fwd(const RopeArgs& a, hipStream_t s) { return a.n == 0 ? hipSuccess : by_type<false>(a, s); }
hipError_t launch_rope_bwd(const RopeArgs& a, hipStream_t s) { return by_type<true>(a, s); }

}  // namespace coset
