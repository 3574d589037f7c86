// kv_cache.hip -- rows of the E8 key/value cache written and read back
// (format and nearest-point rule: kv_cache.hpp).
//
// One lane holds one block of 8 coordinates; the 4 to 32 lanes of a vector
// find its largest magnitude with butterflies.  A workgroup takes one head of
// the keys or the values (blockIdx.y) and 256 / lanes-per-vector tokens, so
// that the values' words of four neighbouring tokens, 16 bytes, leave in the
// same store instruction.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_cache.hpp"
#include "vec_io.hpp"

namespace coset {

namespace {

constexpr int kThreads = 256;

// The word offset of block b of row (page, off, head) and the row's scale.
template <int BITS>
__device__ __forceinline__ int64_t kv_word(const KvCache& c, bool value, int64_t row_base, uint32_t off, int b)
{
    constexpr int W = BITS / 4;
    const int nb = c.dim >> 3;
    const int64_t page = row_base * nb * W;
    return value ? page + ((int64_t)((off >> 2) * nb + b) * 4 + (off & 3)) * W : page + ((int64_t)off * nb + b) * W;
}

template <int BITS, int DT, int GW>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(KvRowsArgs a)
{
    const int lane = threadIdx.x % GW;
    const int64_t t = (int64_t)blockIdx.x * (kThreads / GW) + threadIdx.x / GW;
    const bool value = blockIdx.y & 1;
    const uint32_t head = blockIdx.y >> 1;
    const int nb = a.c.dim >> 3;
    const bool mine = t < a.n && lane < nb;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    int64_t slot = -1;
    if (mine) {
        slot = a.slots[t];
        const int64_t at = t * (value ? a.v_tok : a.k_tok) + head * (value ? a.v_head : a.k_head) + 8 * lane;
        load_n<DT, 8>(value ? a.v : a.k, at, a.vec, x);
    }
    // the largest magnitude as bits: a NaN is above infinity there
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < GW; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    uint32_t scale = kv_scale_bits<BITS>(__uint_as_float(top));
    float beta = __uint_as_float(scale << 16);
    const bool fine = beta > 0.f;   // neither zero nor NaN
    if (!fine) {
        beta = 1.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
    }
    uint32_t w[BITS / 4];
    kv_nearest<BITS>(x, beta, __fdiv_rn(1.f, beta), w);
    if (!mine || slot < 0 || slot >= (int64_t)a.c.pages * a.c.page_size) return;
    const uint32_t page = u32div((uint32_t)slot, a.c.page_div), off = (uint32_t)slot - page * a.c.page_size;
    const int64_t base = ((int64_t)page * a.c.heads + head) * a.c.page_size;
    uint32_t* dst = (value ? a.c.v : a.c.k) + kv_word<BITS>(a.c, value, base, off, lane);
    if constexpr (BITS == 4)
        *dst = w[0];
    else
        *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    if (lane == 0) reinterpret_cast<uint16_t*>(a.c.scales + base + off)[value ? 1 : 0] = (uint16_t)scale;
}

template <int BITS, int DT, int GW>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(KvRowsArgs a)
{
    const int lane = threadIdx.x % GW;
    const int64_t t = (int64_t)blockIdx.x * (kThreads / GW) + threadIdx.x / GW;
    const bool value = blockIdx.y & 1;
    const uint32_t head = blockIdx.y >> 1;
    if (t >= a.n || lane >= (a.c.dim >> 3)) return;
    const int64_t slot = a.slots[t];
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (slot >= 0 && slot < (int64_t)a.c.pages * a.c.page_size) {
        const uint32_t page = u32div((uint32_t)slot, a.c.page_div), off = (uint32_t)slot - page * a.c.page_size;
        const int64_t base = ((int64_t)page * a.c.heads + head) * a.c.page_size;
        const uint32_t* src = (value ? a.c.v : a.c.k) + kv_word<BITS>(a.c, value, base, off, lane);
        uint32_t w[BITS / 4];
        if constexpr (BITS == 4) {
            w[0] = *src;
        } else {
            const uint2 u = *reinterpret_cast<const uint2*>(src);
            w[0] = u.x;
            w[1] = u.y;
        }
        const uint32_t both = a.c.scales[base + off];
        const float beta = __uint_as_float(value ? both & 0xffff0000u : both << 16);
        kv_point<BITS>(w, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= beta;
    }
    store_n<DT, 8>(value ? a.v_out : a.k_out, (t * a.c.heads + head) * (int64_t)a.c.dim + 8 * lane, x);
}

template <int BITS, int DT, int GW, bool WRITE>
hipError_t launch(const KvRowsArgs& a, hipStream_t s)
{
    const dim3 grid((unsigned)((a.n + kThreads / GW - 1) / (kThreads / GW)), 2 * a.c.heads);
    if constexpr (WRITE)
        hipLaunchKernelGGL((kv_write_kernel<BITS, DT, GW>), grid, dim3(kThreads), 0, s, a);
    else
        hipLaunchKernelGGL((kv_read_kernel<BITS, DT, GW>), grid, dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

template <int BITS, int DT, bool WRITE>
hipError_t by_width(const KvRowsArgs& a, hipStream_t s)
{
    const int nb = a.c.dim / 8;
    if (nb <= 4) return launch<BITS, DT, 4, WRITE>(a, s);
    if (nb <= 8) return launch<BITS, DT, 8, WRITE>(a, s);
    if (nb <= 16) return launch<BITS, DT, 16, WRITE>(a, s);
    return launch<BITS, DT, 32, WRITE>(a, s);
}

template <bool WRITE>
hipError_t by_type(const KvRowsArgs& a, hipStream_t s)
{
    if (a.n == 0) return hipSuccess;
    const bool four = a.c.bits == 4;
    switch (a.dtype) {
    case DT_F32: return four ? by_width<4, DT_F32, WRITE>(a, s) : by_width<8, DT_F32, WRITE>(a, s);
    case DT_BF16: return four ? by_width<4, DT_BF16, WRITE>(a, s) : by_width<8, DT_BF16, WRITE>(a, s);
    default: return four ? by_width<4, DT_F16, WRITE>(a, s) : by_width<8, DT_F16, WRITE>(a, s);
    }
}

}  // namespace

hipError_t launch_kv_write(const KvRowsArgs& a, hipStream_t s) { return by_type<true>(a, s); }
hipError_t launch_kv_read(const KvRowsArgs& a, hipStream_t s) { return by_type<false>(a, s); }

}  // namespace coset
