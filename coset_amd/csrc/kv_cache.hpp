// kv_cache.hpp -- keys and values kept as points of E8 (kv_cache.hip writes
// and reads them, kv_attention.hip attends over them).
//
// A head's vector x of D values is one bf16 scale beta and D / 8 points
// lambda of E8 = D8 + {0, 1/2} (1, ..., 1), x_hat = beta lambda.  With C a
// little below 7 (4 bits) or 127 (8 bits) and beta = max|x| / C rounded up,
// the nearest point's coordinates are c_j + h / 2 with c_j in [-8, 7] or
// [-128, 127] and one h in {0, 1} for all eight.  sum c_j is even, so the
// lowest bit of c_7 follows from the others and its place holds h: a block
// takes exactly 8 * BITS bits, and is read back without a table.
//
//   field j of a block (BITS bits, from the lowest): n_j = c_j + 2^(BITS-1),
//   the lowest bit of n_7 replaced by h
//   k       [pages, kv heads, page size, D/8, w]        uint32, w = BITS / 4
//   v       [pages, kv heads, page size / 4, D/8, 4, w] uint32
//   scales  [pages, kv heads, page size, 2]             bf16, key's and value's
//
// Values hold four tokens' words of a block side by side: the attention's
// second product sums over tokens, so a lane wants several tokens of the
// same coordinates (one 16- or 32-byte load), while its first product sums
// over coordinates and wants whole keys.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "codec_kernels.hpp"
#include "fastdiv.hpp"

namespace coset {

struct KvCache {
    uint32_t* k;
    uint32_t* v;
    uint32_t* scales;   // one word per row: key's bf16 in the low half, value's in the high
    uint32_t pages, page_size, heads;
    int dim, bits;
    U32Div page_div;
};

struct KvRowsArgs {
    KvCache c;
    const int64_t* slots;   // [n] rows page * page_size + offset; outside the cache: skipped (write), zeros (read)
    int64_t n;
    const void* k;          // write: [n, heads, dim], strides in elements
    const void* v;
    int64_t k_tok, k_head, v_tok, v_head;
    int vec;                // write: 16-byte loads (pointers and strides allow them)
    void* k_out;            // read: [n, heads, dim] contiguous
    void* v_out;
    int dtype;
};

hipError_t launch_kv_write(const KvRowsArgs& a, hipStream_t s);
hipError_t launch_kv_read(const KvRowsArgs& a, hipStream_t s);

constexpr float kKvSmallest = 0x1p-64f;   // vectors below are stored as zeros
constexpr float kKvLargest = 0x1p64f;     // vectors above (or not finite) read back as NaN

template <int BITS>
__host__ __device__ constexpr float kv_top()
{
    return BITS == 4 ? 7.f - 0x1p-19f : 127.f - 0x1p-15f;
}

// beta for a vector whose largest magnitude is amax: amax / C rounded up to
// bf16, so that no quotient leaves (-C, C) after its rounding (C is 4 or more
// ulps below 7 and 127, two roundings cost one).
template <int BITS>
__device__ __forceinline__ uint32_t kv_scale_bits(float amax)
{
    if (amax < kKvSmallest) return 0u;
    if (!(amax <= kKvLargest)) return 0x7fc0u;
    return (__float_as_uint(__fdiv_rn(amax, kv_top<BITS>())) + 0xffffu) >> 16;
}

// The E8 point nearest to x / beta, packed.  f_j = round(x_j / beta) and the
// remainders r_j = x_j - beta f_j (exact: beta f_j has 15 bits and |r_j| <=
// beta / 2) give both cosets' nearest points: integers f, moved at the largest |r| where
// their sum is odd, and halves f - (r < 0) + 1/2, whose distances are beta/2
// - |r|, moved at the smallest |r|.  The squared distances differ by
//   sum (beta/2 - |r|)^2 - r^2 = beta (2 beta - sum |r|)
// and a move at distance e adds beta^2 - 2 beta e, so the choice needs the
// sum, the largest and the smallest |r| only.  Equal distances go to the
// integers, equal remainders to the first coordinate.
template <int BITS>
__device__ __forceinline__ void kv_nearest(const float (&x)[8], float beta, float inv, uint32_t (&w)[BITS / 4])
{
    float r[8], a[8];
    int c[8];
    int sum = 0, neg = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float f = rintf(div_by_recip<2>(x[j], beta, inv));
        r[j] = fmaf(-f, beta, x[j]);
        a[j] = fabsf(r[j]);
        c[j] = (int)f;
        sum ^= c[j];
        neg ^= r[j] < 0.f ? 1 : 0;
    }
    const float s = __fadd_rn(__fadd_rn(__fadd_rn(a[0], a[4]), __fadd_rn(a[2], a[6])),
                              __fadd_rn(__fadd_rn(a[1], a[5]), __fadd_rn(a[3], a[7])));
    const float most = fmaxf(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])), fmaxf(fmaxf(a[4], a[5]), fmaxf(a[6], a[7])));
    const float least = fminf(fminf(fminf(a[0], a[1]), fminf(a[2], a[3])), fminf(fminf(a[4], a[5]), fminf(a[6], a[7])));
    const bool odd_f = sum & 1, odd_g = (sum ^ neg) & 1;
    const float lhs = __fadd_rn(__fsub_rn(2.f * beta, s), odd_g ? 2.f * least : 0.f);
    const float rhs = odd_f ? __fsub_rn(beta, 2.f * most) : 0.f;
    const bool half = lhs < rhs;
    const float target = half ? least : most;
    bool move = half ? odd_g : odd_f;
    constexpr int kBias = 1 << (BITS - 1);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const bool down = r[j] < 0.f;
        c[j] += kBias - ((half && down) ? 1 : 0);
        const bool hit = move && a[j] == target;
        c[j] += hit ? (down == half ? 1 : -1) : 0;
        move = move && !hit;
    }
    c[7] = (c[7] & ~1) | (half ? 1 : 0);
    constexpr int kPer = 32 / BITS;
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) {
        uint32_t u = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) u |= (uint32_t)c[i * kPer + j] << (BITS * j);
        w[i] = u;
    }
}

// A block's coordinates.
template <int BITS>
__device__ __forceinline__ void kv_point(const uint32_t (&w)[BITS / 4], float (&x)[8])
{
    constexpr int kPer = 32 / BITS;
    constexpr uint32_t kLow = BITS == 4 ? 0x11111111u : 0x01010101u;
    const uint32_t top = w[BITS / 4 - 1];
    const uint32_t h = (top >> (32 - BITS)) & 1u;
    uint32_t all = w[0];
    if constexpr (BITS == 8) all ^= w[1];
    const uint32_t odd = __popc(all & kLow) & 1u;   // parity of the seven low bits and h
    const uint32_t fixed = top ^ (odd << (32 - BITS));   // h xor (parity of the seven xor h)
    const float bias = 0.5f * (float)h - (float)(1 << (BITS - 1));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t u = j / kPer == BITS / 4 - 1 ? fixed : w[j / kPer];
        x[j] = (float)((u >> (BITS * (j % kPer))) & ((1u << BITS) - 1)) + bias;
    }
}

}  // namespace coset
