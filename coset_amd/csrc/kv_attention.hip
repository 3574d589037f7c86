// kv_attention.hip -- attention of new tokens over the E8 key/value cache, in
// one pass over the cached words.
//
//   s_t = scale beta_t (q . lambda_t),  out = sum_t e^{s_t} beta'_t lambda'_t / sum_t e^{s_t}
//
// for the seen tokens t, lambda the key's and lambda' the value's points.
// Points are small half-integers, exact in fp16, so both products run on the
// fp16 matrix cores on the points alone and the scales meet the scores in
// fp32.  A workgroup of four waves takes 16 * NR query rows (tokens x the
// heads that share a key head) of one key head; a wave takes 32 tokens a step:
//
//   S^T[token, row]  = K Q^T   16x16x32, A: a lane's blocks of one key, B: the query rows
//   O^T[dim, row]   += V^T P^T 16x16x32, A: one coordinate of 8 values, B: 8 weights of a row
//
// S^T leaves a lane with 4 + 4 tokens of one row: exactly what the second
// product's B operand wants when its 8 tokens are numbered that way, so the
// weights go from accumulator to operand without leaving the lane, and a
// row's maximum, sum and rescaling are the lane's own.
//
// Weights.  w_t = e^{s_t} beta'_t is rounded to fp16 (11 bits; two fp16 parts
// for fp16 and fp32 calls), relative to 2^M with M such that the largest
// weight of the row so far lies between 2^9 and 2^15; M moves only when a
// weight would pass 2^14, which after the first steps is rare.  Weights down
// to 2^-24 keep a value, 33 or more binary orders below the largest.  M counts beta',
// so that one value of a small weight and a large scale does not push the
// others out of fp16's range.  Sums are fp32.
//
// Work.  The (sequence, key head, row tile) segments' steps of 128 tokens
// form one line; each workgroup takes an equal run of it.  A segment that
// falls to several workgroups is joined by a second kernel from their
// unnormalised rows.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_attention.hpp"
#include "vec_io.hpp"

namespace coset {

namespace {

typedef _Float16 half8_kv __attribute__((ext_vector_type(8)));
typedef _Float16 half2_kv __attribute__((ext_vector_type(2)));
typedef float f32x4_kv __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_kv __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kTile = 32;                   // tokens of a wave's step
constexpr int kStep = kTile * kWaves;       // tokens of a workgroup's step
constexpr float kNone = -1e30f;             // M of a row that has seen nothing
constexpr float kLog2e = 1.44269504088896340736f;

// Tables that no kernel of the call writes, read through the scalar cache
// where the index is the same in all lanes.
typedef const __attribute__((address_space(4))) int32_t* ConstInts;
__device__ __forceinline__ ConstInts constant(const int32_t* p) { return (ConstInts)(uintptr_t)p; }

// log2 of the largest weight with respect to M after a move, and the weight at which the next move is due
constexpr float kSettle = 9.f, kDue = 0x1p14f;

// One descriptor a workgroup: the parts of the segment that begins in it and
// goes on in the next ones (0: none).
struct Desc {
    int parts;       // this workgroup's and those of the following ones
    int row0;        // first row of the row tile
    int rows;        // rows in it
    int token0;      // first query token of the sequence
    int head;        // key head
    int pad[3];
};

struct Work {
    int steps;       // of 128 tokens in a segment
    int tiles;       // row tiles
    int units;       // steps * tiles * key heads
};

struct Seq {
    int token0, tokens, length;
};

__device__ __forceinline__ Seq seq_of(const KvAttentionArgs& a, int b)
{
    Seq s;
    if (a.starts) {
        // starts outside [0, n], or in falling order: no tokens
        const int lo = constant(a.starts)[b], hi = constant(a.starts)[b + 1];
        s.token0 = min(max(lo, 0), (int)a.n);
        s.tokens = max(min(max(hi, 0), (int)a.n) - s.token0, 0);
    } else {
        s.tokens = (int)(a.n / a.seqs);
        s.token0 = b * s.tokens;
    }
    s.length = min(max(constant(a.lengths)[b], 0), (int)min((int64_t)a.max_pages * a.c.page_size, (int64_t)0x7fffff00));
    return s;
}

__device__ __forceinline__ Work work_of(const KvAttentionArgs& a, const Seq& s, int rows)
{
    Work w;
    w.steps = max((s.length + kStep - 1) / kStep, 1);
    w.tiles = (s.tokens * a.group + rows - 1) / rows;
    w.units = w.steps * w.tiles * (int)a.c.heads;
    return w;
}

// The A operand of 16 keys: blocks' eight points as 2^k-offset fp16 pairs
// (elements i and i + 4 in register i), value = offset + coordinate with
// offset 24 (4 bits) or 640 (8 bits).
template <int BITS>
constexpr float kOffset = BITS == 4 ? 24.f : 640.f;

__device__ __forceinline__ uint32_t minus(uint32_t u, float off)
{
    const half2_kv o = {(_Float16)off, (_Float16)off};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_kv, u) - o);
}

// Nibble fields sit at bits 6..9 of a half whose exponent is that of [16, 32):
// 16 + n + h / 2.  Bytes sit at bits 1..8 of one whose exponent is that of
// [512, 1024): 512 + n + h / 2.
template <int I>
__device__ __forceinline__ uint32_t nibbles(uint32_t u, uint32_t base)
{
    const uint32_t s = I == 0 ? u << 6 : I == 1 ? u << 2 : I == 2 ? u >> 2 : u >> 6;
    return (s & 0x03c003c0u) | base;
}

template <int BITS, bool CENTER>
__device__ __forceinline__ void key_operand(const uint32_t* w, uint32_t (&r)[4])
{
    if constexpr (BITS == 4) {
        const uint32_t base = ((uint32_t)__builtin_amdgcn_sbfe((int)w[0], 28, 1) & 0x00200020u) | 0x4c004c00u;
        r[0] = nibbles<0>(w[0], base);
        r[1] = nibbles<1>(w[0], base);
        r[2] = nibbles<2>(w[0], base);
        // n_7's lowest bit, at 22 here: h there, xor the parity of the word's lowest bits
        r[3] = nibbles<3>(w[0], base) ^ ((uint32_t)__popc(w[0] & 0x11111111u) << 22 & 0x00400000u);
    } else {
        const uint32_t h = (w[1] >> 24) & 1u;
        const uint32_t base = 0x60006000u | h | (h << 16);
        const uint32_t hi = w[1] ^ ((uint32_t)__popc((w[0] ^ w[1]) & 0x01010101u) << 31 >> 7);
        // byte i of the low word and of the high word
        r[0] = (__builtin_amdgcn_perm(hi, w[0], 0x0c040c00u) << 1) | base;
        r[1] = (__builtin_amdgcn_perm(hi, w[0], 0x0c050c01u) << 1) | base;
        r[2] = (__builtin_amdgcn_perm(hi, w[0], 0x0c060c02u) << 1) | base;
        r[3] = (__builtin_amdgcn_perm(hi, w[0], 0x0c070c03u) << 1) | base;
    }
    if constexpr (CENTER)
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = minus(r[i], kOffset<BITS>);
}

// Coordinates of one block of two tokens as centred fp16 pairs: register e
// holds coordinate e (E = 8), or e + 4 * upper (E = 4).
template <int BITS, int E>
__device__ __forceinline__ void value_pair(const uint32_t* a, const uint32_t* b, bool upper, uint32_t (&r)[E])
{
    if constexpr (BITS == 4) {
        const uint32_t lo = __builtin_amdgcn_perm(b[0], a[0], 0x05040100u);
        const uint32_t hi = __builtin_amdgcn_perm(b[0], a[0], 0x07060302u);
        uint32_t z = lo ^ hi;   // lowest bits of the fields, at 0, 4, 8, 12 of each half
        z ^= z << 8;
        z ^= z << 4;
        const uint32_t base = 0x4c004c00u | ((hi >> 7) & 0x00200020u);
        const uint32_t fixed = hi ^ (z & 0x10001000u);
        if constexpr (E == 8) {
            r[0] = nibbles<0>(lo, base);
            r[1] = nibbles<1>(lo, base);
            r[2] = nibbles<2>(lo, base);
            r[3] = nibbles<3>(lo, base);
            r[4] = nibbles<0>(fixed, base);
            r[5] = nibbles<1>(fixed, base);
            r[6] = nibbles<2>(fixed, base);
            r[7] = nibbles<3>(fixed, base);
        } else {
            const uint32_t u = upper ? fixed : lo;
            r[0] = nibbles<0>(u, base);
            r[1] = nibbles<1>(u, base);
            r[2] = nibbles<2>(u, base);
            r[3] = nibbles<3>(u, base);
        }
    } else {
        const uint32_t base = 0x60006000u | ((a[1] >> 24) & 1u) | ((b[1] >> 8) & 0x00010000u);
        const uint32_t ha = a[1] ^ ((uint32_t)__popc((a[0] ^ a[1]) & 0x01010101u) << 31 >> 7);
        const uint32_t hb = b[1] ^ ((uint32_t)__popc((b[0] ^ b[1]) & 0x01010101u) << 31 >> 7);
        const uint32_t la = E == 4 && upper ? ha : a[0], lb = E == 4 && upper ? hb : b[0];
        r[0] = (__builtin_amdgcn_perm(lb, la, 0x0c040c00u) << 1) | base;
        r[1] = (__builtin_amdgcn_perm(lb, la, 0x0c050c01u) << 1) | base;
        r[2] = (__builtin_amdgcn_perm(lb, la, 0x0c060c02u) << 1) | base;
        r[3] = (__builtin_amdgcn_perm(lb, la, 0x0c070c03u) << 1) | base;
        if constexpr (E == 8) {
            r[4] = (__builtin_amdgcn_perm(hb, ha, 0x0c040c00u) << 1) | base;
            r[5] = (__builtin_amdgcn_perm(hb, ha, 0x0c050c01u) << 1) | base;
            r[6] = (__builtin_amdgcn_perm(hb, ha, 0x0c060c02u) << 1) | base;
            r[7] = (__builtin_amdgcn_perm(hb, ha, 0x0c070c03u) << 1) | base;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) r[e] = minus(r[e], kOffset<BITS>);
}

// What a wave loads for 16 tokens: a lane's blocks of one key, four tokens'
// words of its block (or two blocks) of the values, four tokens' scales.  The
// row is wave-uniform, a lane's place in it is fixed.
template <int DP, int BITS>
struct Words {
    static constexpr int W = BITS / 4;
    static constexpr int C = DP / 32;               // 32-coordinate chunks: a lane's blocks of a key
    static constexpr int B = DP == 256 ? 2 : 1;     // a lane's blocks of the values
    static constexpr int KL = C * W == 2 ? 1 : C * W / 4;   // loads of a lane's keys
    uint32_t k_at[KL], v_at[B], s_at;               // byte offsets from the row
    int row_bytes;

    __device__ __forceinline__ void init(const KvCache& c, int lane)
    {
        const int nb = c.dim >> 3, g = lane >> 4, m = lane & 15;
        row_bytes = 4 * nb * W;
        if constexpr (C * W == 2) {
            k_at[0] = m * row_bytes + 8 * min(g, nb / 2 - 1);
        } else {
#pragma unroll
            for (int i = 0; i < KL; ++i) k_at[i] = m * row_bytes + 16 * min(g * KL + i, nb * W / 4 - 1);
        }
#pragma unroll
        for (int b = 0; b < B; ++b) v_at[b] = 4 * g * row_bytes + 16 * W * min(DP == 64 ? m & 7 : 16 * b + m, nb - 1);
        s_at = 16 * g;
    }

    __device__ __forceinline__ void keys(const KvCache& c, int64_t row, uint32_t (&k)[C * W]) const
    {
        const char* p = reinterpret_cast<const char*>(c.k) + row * row_bytes;
        if constexpr (C * W == 2) {
            const uint2 u = *reinterpret_cast<const uint2*>(p + k_at[0]);
            k[0] = u.x;
            k[1] = u.y;
        } else {
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                const u32x4_kv u = *reinterpret_cast<const u32x4_kv*>(p + k_at[i]);
#pragma unroll
                for (int j = 0; j < 4; ++j) k[4 * i + j] = u[j];
            }
        }
    }

    __device__ __forceinline__ void values(const KvCache& c, int64_t row, uint32_t (&v)[B][4 * W]) const
    {
        const char* p = reinterpret_cast<const char*>(c.v) + row * row_bytes;
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const u32x4_kv u = *reinterpret_cast<const u32x4_kv*>(p + v_at[b] + 16 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[b][4 * i + j] = u[j];
            }
    }

    __device__ __forceinline__ void scales(const KvCache& c, int64_t row, uint32_t (&sc)[4]) const
    {
        const u32x4_kv u = *reinterpret_cast<const u32x4_kv*>(reinterpret_cast<const char*>(c.scales) + row * 4 + s_at);
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[j] = u[j];
    }
};

__device__ __forceinline__ float over_groups_max(float v)
{
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}

__device__ __forceinline__ float over_groups_sum(float v)
{
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// Which of the tokens place .. place + 3 a row sees: those below its limit
// and, with a mask, the drafted ones whose bits its row of the mask sets.
__device__ __forceinline__ uint32_t seen_of(const KvAttentionArgs& a, const Seq& sq, int limit, int own, int place)
{
    uint32_t seen = 0;
    const int ctx = sq.length - sq.tokens;
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
        const int at = place + i, d = at - ctx;
        bool on = at < limit;
        if (a.mask && !on && own >= 0 && at < sq.length && d >= 0 && d < 64 * a.mask_words)
            on = (a.mask[(int64_t)own * a.mask_words + (d >> 6)] >> (d & 63)) & 1;
        seen |= on ? 1u << i : 0u;
    }
    return seen;
}

template <int DT>
__device__ __forceinline__ void load_query(const KvAttentionArgs& a, int64_t at, float (&x)[8])
{
    load_n<DT, 8>(a.q, at, a.vec, x);
}

// DP: dim padded to 64, 128 or 256; NR: 16-row tiles; QS: queries in two fp16
// parts; PS: weights in two.
template <int DP, int BITS, int NR, int DT, bool QS, bool PS, int OCC>
__global__ void __launch_bounds__(kThreads, OCC) kv_attention_kernel(KvAttentionArgs a, int most_parts)
{
    using T = Words<DP, BITS>;
    constexpr int C = T::C, W = T::W;
    constexpr int E = DP == 64 ? 4 : 8;          // a lane's coordinates of a value block
    constexpr int NT = DP / 16;                  // accumulator tiles of a row tile
    constexpr int kRows = 16 * NR;
    constexpr int kPitch = DP + 4;
    __shared__ __align__(16) float sh_o[kWaves][16 * kPitch];
    __shared__ float sh_m[kWaves][kRows], sh_l[kWaves][kRows];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    T words;
    words.init(a.c, lane);
    // neighbouring runs on one XCD (workgroups go to the 8 XCDs in turn)
    const int id = (int)(blockIdx.x & 7) * (gridDim.x >> 3) + (int)(blockIdx.x >> 3);

    // the line of units: its length, this workgroup's run and where it begins
    int total = 0;
    for (int b0 = 0; b0 < a.seqs; b0 += 64) {
        int u = b0 + lane < a.seqs ? work_of(a, seq_of(a, b0 + lane), kRows).units : 0;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) u += __shfl_xor(u, o, 64);
        total += u;
    }
    total = __builtin_amdgcn_readfirstlane(total);
    const int run = (total + (int)gridDim.x - 1) / (int)gridDim.x;
    int unit = id * run;
    const int end = min(unit + run, total);
    Desc* descs = reinterpret_cast<Desc*>(a.workspace);
    float* part_ml = a.workspace + (int64_t)gridDim.x * (sizeof(Desc) / 4);
    float* part_o = part_ml + (int64_t)gridDim.x * 2 * kRows * 2;
    if (most_parts > 1 && threadIdx.x == 0 && unit >= end) descs[id].parts = 0;
    if (unit >= end) return;
    int b = 0, before = 0;
    for (int b0 = 0; b0 < a.seqs; b0 += 64) {
        const int u = b0 + lane < a.seqs ? work_of(a, seq_of(a, b0 + lane), kRows).units : 0;
        int sum = u;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int up = __shfl_up(sum, o, 64);
            sum += lane >= o ? up : 0;
        }
        const uint64_t past = __ballot(before + sum > unit);
        if (past) {
            const int first = __ffsll((unsigned long long)past) - 1;
            b = b0 + first;
            before += __shfl(sum - u, first, 64);
            break;
        }
        before += __shfl(sum, 63, 64);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    before = __builtin_amdgcn_readfirstlane(before);
    Seq sq = seq_of(a, b);
    Work wk = work_of(a, sq, kRows);
    int seg = (unit - before) / wk.steps, step = (unit - before) % wk.steps;
    if (most_parts > 1 && threadIdx.x == 0) descs[id].parts = 0;
    if (seg >= wk.tiles * (int)a.c.heads) return;   // starts that overlap so far that the line's length wrapped

    while (unit < end) {
        const int count = min(wk.steps - step, end - unit);
        const int kh = seg / wk.tiles, tile = seg % wk.tiles;
        const int row0 = tile * kRows, rows = min(sq.tokens * a.group - row0, kRows);
        const int ctx = sq.length - sq.tokens;
        const int t_first = u32div((uint32_t)row0, a.group_div);
        const int t_last = u32div((uint32_t)(row0 + rows - 1), a.group_div);

        // the query rows
        uint32_t q_hi[NR][C][4], q_lo[NR][QS ? C : 1][4];
        float q_scale[NR], q_bias[NR];
        int limit[NR], own[NR];     // a row sees tokens below limit; own: its query token
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int row = 16 * r + n;
            const bool on = row < rows;
            const uint32_t t = u32div((uint32_t)(row0 + row), a.group_div);
            const int hq = kh * a.group + (row0 + row - (int)t * a.group);
            own[r] = on ? sq.token0 + (int)t : -1;
            limit[r] = on ? (a.mask ? ctx : min(sq.length, ctx + (int)t + 1)) : 0;
            float x[C][8];
            float top = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int block = C * g + c;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[c][j] = 0.f;
                if (on && block < (a.c.dim >> 3))
                    load_query<DT>(a, (int64_t)own[r] * a.q_tok + hq * a.q_head + 8 * block, x[c]);
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[c][j]));
            }
            top = over_groups_max(top);
            // times 2^k, which brings the row's largest value to [2^10, 2^11)
            const int e = max((int)(__float_as_uint(top) >> 23), 20);
            const float up = copysignf(__uint_as_float((uint32_t)(264 - e) << 23), a.scale);
            // above zero, so that a hidden token's score stays at minus infinity
            q_scale[r] = fmaxf(fabsf(a.scale) * __uint_as_float((uint32_t)(e - 10) << 23), 0x1p-126f);
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float u = x[c][i] * up, v = x[c][i + 4] * up;
                    q_hi[r][c][i] = pack2<DT_F16>(u, v);
                    float hu, hv;
                    unpack2<DT_F16>(q_hi[r][c][i], hu, hv);
                    sum += hu + hv;
                    if constexpr (QS) q_lo[r][c][i] = pack2<DT_F16>(u - hu, v - hv);
                }
            }
            q_bias[r] = QS ? 0.f : -kOffset<BITS> * over_groups_sum(sum);
        }

        float M[NR], l[NR];
        f32x4_kv o[NR][NT];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            M[r] = kNone;
            l[r] = 0.f;
#pragma unroll
            for (int j = 0; j < NT; ++j) o[r][j] = f32x4_kv{0.f, 0.f, 0.f, 0.f};
        }

        // tokens that any row of the tile may see, and those that all see
        const int reach = a.mask ? sq.length : min(sq.length, ctx + t_last + 1);
        const int all = a.mask ? ctx : ctx + t_first + 1;
        const ConstInts pages = constant(a.table + (int64_t)b * a.table_stride);
        auto row_of = [&](int token) -> int64_t {
            const uint32_t i = u32div((uint32_t)token, a.c.page_div);
            const uint32_t page = min((uint32_t)max(pages[min((int)i, a.max_pages - 1)], 0), a.c.pages - 1);
            return ((int64_t)page * a.c.heads + kh) * a.c.page_size + (token - i * a.c.page_size);
        };

        int token = (step * kWaves + wave) * kTile;
        const int stop = min((step + count) * kStep, reach);
        // one set of registers: the next keys are loaded behind the scores'
        // product, the next values behind the second one, so that each has
        // about half a step to arrive
        uint32_t kw[2][C * W], vw[2][T::B][4 * W], sc[2][4];
        int64_t at[2];
        if (token < stop) {
            at[0] = row_of(token);
            at[1] = row_of(token + 16 < reach ? token + 16 : token);
#pragma unroll
            for (int h = 0; h < 2; ++h) words.keys(a.c, at[h], kw[h]);
#pragma unroll
            for (int h = 0; h < 2; ++h) words.scales(a.c, at[h], sc[h]);
#pragma unroll
            for (int h = 0; h < 2; ++h) words.values(a.c, at[h], vw[h]);
        }
        for (; token < stop; token += kStep) {
            const int ahead = token + kStep < stop ? token + kStep : token;
            at[0] = row_of(ahead);
            at[1] = row_of(ahead + 16 < reach ? ahead + 16 : ahead);
            // scores
            f32x4_kv s[2][NR];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int r = 0; r < NR; ++r) s[h][r] = f32x4_kv{q_bias[r], q_bias[r], q_bias[r], q_bias[r]};
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    uint32_t k[4];
                    key_operand<BITS, QS>(&kw[h][c * W], k);
                    const half8_kv ka = __builtin_bit_cast(half8_kv, u32x4_kv{k[0], k[1], k[2], k[3]});
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        s[h][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            ka, __builtin_bit_cast(half8_kv, u32x4_kv{q_hi[r][c][0], q_hi[r][c][1], q_hi[r][c][2], q_hi[r][c][3]}),
                            s[h][r], 0, 0, 0);
                        if constexpr (QS)
                            s[h][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                ka, __builtin_bit_cast(half8_kv, u32x4_kv{q_lo[r][c][0], q_lo[r][c][1], q_lo[r][c][2], q_lo[r][c][3]}),
                                s[h][r], 0, 0, 0);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) words.keys(a.c, at[h], kw[h]);
            // weights
            const bool whole = token + kTile <= all;
            float bk[8], bv[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t u = sc[i >> 2][i & 3];
                bk[i] = __uint_as_float(u << 16);
                // a zero vector's scale as 2^-70 (its points are zeros): no infinity times zero below
                bv[i] = __uint_as_float(max(u & 0xffff0000u, 0x1c800000u));
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) words.scales(a.c, at[h], sc[h]);
            uint32_t p_hi[NR][4], p_lo[NR][4];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float u[8], w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] = s[i >> 2][r][i & 3] * bk[i];
                uint32_t seen = 0xffu;
                if (!whole) {
                    seen = seen_of(a, sq, limit[r], own[r], token + 4 * g) | seen_of(a, sq, limit[r], own[r], token + 16 + 4 * g) << 4;
#pragma unroll
                    for (int i = 0; i < 8; ++i) u[i] = seen >> i & 1u ? u[i] : -INFINITY;
                }
                float sum = 0.f, top = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(u[i], q_scale[r], -M[r]));
                    sum += p;
                    w[i] = p * bv[i];
                }
                if (!whole) {   // zero times a NaN scale
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[i] = seen >> i & 1u ? w[i] : 0.f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, w[i]);
                if (__any(top > kDue)) {
                    float most = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 8; ++i) most = fmaxf(most, fmaf(u[i], q_scale[r], __builtin_amdgcn_logf(bv[i])));
                    const float to = fmaxf(M[r], over_groups_max(most) - kSettle);
                    const float f = __builtin_amdgcn_exp2f(M[r] - to);
                    M[r] = to;
                    l[r] *= f;
#pragma unroll
                    for (int j = 0; j < NT; ++j) o[r][j] *= f;
                    sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(u[i], q_scale[r], -to));
                        sum += p;
                        w[i] = seen >> i & 1u ? p * bv[i] : 0.f;
                    }
                }
                l[r] += sum;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p_hi[r][i] = pack2<DT_F16>(w[2 * i], w[2 * i + 1]);
                    if constexpr (PS) {
                        float x, y;
                        unpack2<DT_F16>(p_hi[r][i], x, y);
                        p_lo[r][i] = pack2<DT_F16>(w[2 * i] - x, w[2 * i + 1] - y);
                    }
                }
            }
            // values
#pragma unroll
            for (int blk = 0; blk < T::B; ++blk) {
                uint32_t v[4][E];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    value_pair<BITS, E>(&vw[i >> 1][blk][(i & 1) * 2 * W], &vw[i >> 1][blk][((i & 1) * 2 + 1) * W], n >= 8, v[i]);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const half8_kv va = __builtin_bit_cast(half8_kv, u32x4_kv{v[0][e], v[1][e], v[2][e], v[3][e]});
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        o[r][blk * 8 + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            va, __builtin_bit_cast(half8_kv, u32x4_kv{p_hi[r][0], p_hi[r][1], p_hi[r][2], p_hi[r][3]}),
                            o[r][blk * 8 + e], 0, 0, 0);
                        if constexpr (PS)
                            o[r][blk * 8 + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                va, __builtin_bit_cast(half8_kv, u32x4_kv{p_lo[r][0], p_lo[r][1], p_lo[r][2], p_lo[r][3]}),
                                o[r][blk * 8 + e], 0, 0, 0);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) words.values(a.c, at[h], vw[h]);
        }

        // the four waves' rows
        const bool done = count == wk.steps;
        const int slot = 2 * id + (step == 0 ? 1 : 0);   // a segment's first part, or a later one
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const float sum = over_groups_sum(l[r]);
            if (g == 0) {
                sh_m[wave][16 * r + n] = M[r];
                sh_l[wave][16 * r + n] = sum;
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            float m = sh_m[0][16 * r + n];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) m = fmaxf(m, sh_m[w][16 * r + n]);
            const float f = __builtin_amdgcn_exp2f(M[r] - m);
            float* mine = &sh_o[wave][n * kPitch];
            if constexpr (DP == 64) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 8 * ((4 * g + i) & 7) + 4 * (g >> 1);
                    *reinterpret_cast<f32x4_kv*>(mine + d) =
                        f32x4_kv{o[r][0][i], o[r][1][i], o[r][2][i], o[r][3][i]} * f;
                }
            } else {
#pragma unroll
                for (int blk = 0; blk < T::B; ++blk)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 8; e += 4) {
                            const int d = 128 * blk + 8 * (4 * g + i) + e;
                            *reinterpret_cast<f32x4_kv*>(mine + d) =
                                f32x4_kv{o[r][8 * blk + e][i], o[r][8 * blk + e + 1][i], o[r][8 * blk + e + 2][i],
                                         o[r][8 * blk + e + 3][i]} * f;
                        }
            }
            __syncthreads();
            // 16 rows x DP: a thread takes DP / 16 neighbours of one row in pieces of 8
            const int row = threadIdx.x >> 4;
            const int rr = 16 * r + row;
            float mm = sh_m[0][rr];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) mm = fmaxf(mm, sh_m[w][rr]);
            float ll = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) ll += sh_l[w][rr] * __builtin_amdgcn_exp2f(sh_m[w][rr] - mm);
            if (rr < rows) {
                const uint32_t t = u32div((uint32_t)(row0 + rr), a.group_div);
                const int hq = kh * a.group + (row0 + rr - (int)t * a.group);
                const int64_t at = ((int64_t)sq.token0 + t) * a.heads + hq;
                const float inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
                for (int d = 8 * (threadIdx.x & 15); d < a.c.dim; d += 128) {
                    float x[8];
#pragma unroll
                    for (int j = 0; j < 8; j += 4) {
                        f32x4_kv v = *reinterpret_cast<const f32x4_kv*>(&sh_o[0][row * kPitch + d + j]);
#pragma unroll
                        for (int w = 1; w < kWaves; ++w)
                            v += *reinterpret_cast<const f32x4_kv*>(&sh_o[w][row * kPitch + d + j]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[j + i] = v[i];
                    }
                    if (done) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] *= inv;
                        store_n<DT, 8>(a.out, at * a.c.dim + d, x);
                    } else {
                        store_n<DT_F32, 8>(part_o, ((int64_t)slot * kRows + rr) * DP + d, x);
                    }
                }
                if ((threadIdx.x & 15) == 0) {
                    if (done) {
                        if (a.lse) a.lse[at] = ll > 0.f || ll != ll ? (mm + log2f(ll)) * (1.f / kLog2e) : -INFINITY;
                    } else {
                        part_ml[((int64_t)slot * kRows + rr) * 2] = mm;
                        part_ml[((int64_t)slot * kRows + rr) * 2 + 1] = ll;
                    }
                }
            }
            __syncthreads();
        }
        if (!done && step == 0 && threadIdx.x == 0) {
            Desc d{};
            d.parts = min(1 + (wk.steps - count + run - 1) / run, (int)gridDim.x - id);
            d.row0 = row0;
            d.rows = rows;
            d.token0 = sq.token0;
            d.head = kh;
            descs[id] = d;
        }

        unit += count;
        step = 0;
        if (unit < end && ++seg == wk.tiles * (int)a.c.heads) {
            seg = 0;
            do {
                if (++b >= a.seqs) return;
                sq = seq_of(a, b);
                wk = work_of(a, sq, kRows);
            } while (wk.units == 0);
        }
    }
}

// Joins the parts of the segment that begins in workgroup blockIdx.x: one
// workgroup a row (blockIdx.y), DP / 4 threads across the row, the rest of
// them across the parts.
template <int DP, int NR, int DT>
__global__ void __launch_bounds__(kThreads) kv_join_kernel(KvAttentionArgs a, int blocks)
{
    constexpr int kRows = 16 * NR;
    constexpr int kAcross = DP / 4, kParts = kThreads / kAcross;
    __shared__ __align__(16) float sh_o[kParts][DP];
    __shared__ float sh_m[kParts], sh_l[kParts];
    const Desc d = reinterpret_cast<const Desc*>(a.workspace)[blockIdx.x];
    const int row = blockIdx.y;
    if (d.parts == 0 || row >= d.rows) return;
    const float* part_ml = a.workspace + (int64_t)blocks * (sizeof(Desc) / 4);
    const float* part_o = part_ml + (int64_t)blocks * 2 * kRows * 2;
    const int across = threadIdx.x % kAcross, lot = threadIdx.x / kAcross;
    auto slot = [&](int p) { return (int64_t)(2 * ((int)blockIdx.x + p) + (p == 0 ? 1 : 0)) * kRows + row; };
    float m = kNone;
    for (int p = lot; p < d.parts; p += kParts) m = fmaxf(m, part_ml[slot(p) * 2]);
    if (across == 0) sh_m[lot] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kParts; ++i) m = fmaxf(m, sh_m[i]);
    f32x4_kv o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    for (int p = lot; p < d.parts; p += kParts) {
        const int64_t at = slot(p);
        const float f = __builtin_amdgcn_exp2f(part_ml[at * 2] - m);
        l += part_ml[at * 2 + 1] * f;
        if (4 * across < a.c.dim) o += *reinterpret_cast<const f32x4_kv*>(part_o + at * DP + 4 * across) * f;
    }
    *reinterpret_cast<f32x4_kv*>(&sh_o[lot][4 * across]) = o;
    if (across == 0) sh_l[lot] = l;
    __syncthreads();
    if (lot != 0 || 4 * across >= a.c.dim) return;
#pragma unroll
    for (int i = 1; i < kParts; ++i) {
        o += *reinterpret_cast<const f32x4_kv*>(&sh_o[i][4 * across]);
        l += sh_l[i];
    }
    const bool some = l > 0.f || l != l;
    const float inv = some ? 1.f / l : 0.f;
    const uint32_t t = u32div((uint32_t)(d.row0 + row), a.group_div);
    const int64_t at = ((int64_t)d.token0 + t) * a.heads + d.head * a.group + (d.row0 + row - (int)t * a.group);
    const float x[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    store_n<DT, 4>(a.out, at * a.c.dim + 4 * across, x);
    if (a.lse && across == 0) a.lse[at] = some ? (m + log2f(l)) * (1.f / kLog2e) : -INFINITY;
}

// Waves a SIMD, and so workgroups a CU, that the registers leave room for.
constexpr int waves_of(int pad_dim, int tiles) { return pad_dim == 256 || tiles == 4 ? 1 : tiles == 2 ? 2 : 3; }

template <int DP, int BITS, int NR, int DT>
hipError_t launch(const KvAttentionArgs& a, const KvAttentionPlan& p, hipStream_t s)
{
    constexpr bool QS = DT == DT_F32, PS = DT != DT_BF16;
    constexpr int OCC = waves_of(DP, NR);
    const int64_t most_tokens = (int64_t)a.max_pages * a.c.page_size;
    const int most_parts = (int)((most_tokens + kStep - 1) / kStep);
    hipLaunchKernelGGL((kv_attention_kernel<DP, BITS, NR, DT, QS, PS, OCC>), dim3(p.blocks), dim3(kThreads), 0, s, a, most_parts);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || most_parts <= 1) return e;
    // rows of a tile that can be in use
    const int64_t rows = a.starts ? a.n * a.group : a.n / a.seqs * a.group;
    hipLaunchKernelGGL((kv_join_kernel<DP, NR, DT>), dim3(p.blocks, (unsigned)(rows < 16 * NR ? rows : 16 * NR)),
                       dim3(kThreads), 0, s, a, p.blocks);
    return hipGetLastError();
}

template <int DP, int BITS, int DT>
hipError_t by_tiles(const KvAttentionArgs& a, const KvAttentionPlan& p, hipStream_t s)
{
    if (p.tiles == 1) return launch<DP, BITS, 1, DT>(a, p, s);
    if constexpr (DT != DT_F32 || DP < 256) {
        if (p.tiles == 2) return launch<DP, BITS, 2, DT>(a, p, s);
    }
    if constexpr (DT != DT_F32 && DP < 256) {
        if (p.tiles == 4) return launch<DP, BITS, 4, DT>(a, p, s);
    }
    return hipErrorInvalidValue;
}

template <int DT>
hipError_t by_format(const KvAttentionArgs& a, const KvAttentionPlan& p, hipStream_t s)
{
    const bool four = a.c.bits == 4;
    switch (p.pad_dim) {
    case 64: return four ? by_tiles<64, 4, DT>(a, p, s) : by_tiles<64, 8, DT>(a, p, s);
    case 128: return four ? by_tiles<128, 4, DT>(a, p, s) : by_tiles<128, 8, DT>(a, p, s);
    default: return four ? by_tiles<256, 4, DT>(a, p, s) : by_tiles<256, 8, DT>(a, p, s);
    }
}

}  // namespace

KvAttentionPlan kv_attention_plan(int64_t n, int seqs, int heads, int kv_heads, int dim, int bits, int dtype,
                                  int64_t max_tokens)
{
    (void)bits;
    KvAttentionPlan p{};
    p.pad_dim = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
    const int64_t rows = (n + seqs - 1) / seqs * (heads / kv_heads);
    const int most = dtype == DT_F32 ? (p.pad_dim == 256 ? 1 : 2) : (p.pad_dim == 256 ? 2 : 4);
    p.tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    if (p.tiles > most) p.tiles = most;
    // workgroups that fit the chip at once, fewer where the steps are fewer
    const int64_t tiles = (n * (heads / kv_heads) + 16 * p.tiles - 1) / (16 * p.tiles) + seqs;
    const int64_t steps = (max_tokens + kStep - 1) / kStep;
    const int64_t units = p.units = tiles * kv_heads * (steps > 0 ? steps : 1);
    const int64_t fit = 256 * waves_of(p.pad_dim, p.tiles);
    p.blocks = (int)(units < fit ? (units + 7) / 8 * 8 : fit);
    if (p.blocks < 8) p.blocks = 8;
    const int64_t r = 16 * p.tiles;
    p.workspace_floats = (int64_t)p.blocks * ((int64_t)sizeof(Desc) / 4 + 2 * r * 2 + 2 * r * p.pad_dim);
    return p;
}

hipError_t launch_kv_attention(const KvAttentionArgs& a, const KvAttentionPlan& p, hipStream_t s)
{
    switch (a.dtype) {
    case DT_F32: return by_format<DT_F32>(a, p, s);
    case DT_BF16: return by_format<DT_BF16>(a, p, s);
    default: return by_format<DT_F16>(a, p, s);
    }
}

}  // namespace coset
