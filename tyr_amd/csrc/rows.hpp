// What the kernels that keep rows of bf16 in registers share (RMS norm, layer norm): pieces of 8 elements, sums over the lanes of a row,
// rows whose squares f32 does not hold, rows as buffers.
#pragma once
#include "common.hpp"
#include <type_traits>
#include <utility>

namespace tyr {
namespace row_ops {
__device__ __forceinline__ void unpack8(u32x4 v, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = bf16_lo(v[i]); f[2 * i + 1] = bf16_hi(v[i]); }
}
__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack_bf16(f[2 * i], f[2 * i + 1]);
    return v;
}

// f(0), f(1), ... f(N - 1), each with its own type: an array that they index is registers from the start.  (As loops, beside the branch for rows
// beyond f32, the weights became one block of registers, and the second piece was asked for when the first was there.)
template <int... I, class F>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F f) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F>
__device__ __forceinline__ void each(F f) { each_of(std::make_integer_sequence<int, N>{}, f); }

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// Over groups of LANES lanes, the same bits in every lane of a group.  The steps within 16 lanes are moves of the vector unit
// (quads, halves of a row and rows mirrored); __shfl_xor goes through LDS.
template <int LANES, class F>
__device__ __forceinline__ float over_lanes(float x, F op) {
    if constexpr (LANES >= 2) x = op(x, dpp<0xb1>(x));
    if constexpr (LANES >= 4) x = op(x, dpp<0x4e>(x));
    if constexpr (LANES >= 8) x = op(x, dpp<0x141>(x));
    if constexpr (LANES >= 16) x = op(x, dpp<0x140>(x));
    if constexpr (LANES >= 32) x = op(x, xor16(x));
    if constexpr (LANES >= 64) x = op(x, xor32(x));
    return x;
}
// bf16 holds rows whose squares f32 does not.  Where a row's mean square, eps with it, is outside of [LEAST, infinity), its statistics are
// taken again from h 2^k (and eps 2^2k): y is the same for every k.  Such a row is read twice more, by each of its waves alone: no barrier.
// What the test costs the others: 65536 x 1024 87.7 us without it, 87.9 so; its gradients 89.7, 90.7; 2000 x 4096 16.0, 16.0.
constexpr float LEAST = 0x1p-70f;
__device__ __forceinline__ bool beyond(float mean) {                // or NaN
    return __builtin_bit_cast(uint32_t, mean) - __builtin_bit_cast(uint32_t, LEAST) >= 0x7f800000u - __builtin_bit_cast(uint32_t, LEAST);
}
// of any row of a wave; rows of whole waves by the scalar unit
template <int LPR>
__device__ __forceinline__ bool any_beyond(float mean) {
    if constexpr (LPR == 64) mean = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, mean)));
    else return __builtin_amdgcn_ballot_w64(beyond(mean)) != 0;
    return beyond(mean);
}
// the power of two that brings a number that is not negative to [1, 4), or as near as 2^-126 and 2^100 do
__device__ __forceinline__ float power_for(float most) {
    const int e = min(253, max(27, (int)(__builtin_bit_cast(uint32_t, most) >> 23)));
    return __builtin_bit_cast(float, (uint32_t)(254 - e) << 23);
}

struct Add { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct Max { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };

// Rows as a buffer of `bytes` bytes.  Reads beyond it give 0 and writes beyond it are dropped, without a branch: behind a branch the
// compiler no longer knows which loads and stores are under way and waits for all of them.
constexpr int NOWHERE = 0x40000000, NT = 2;                     // an offset beyond every buffer; cache policy: not kept
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const uint16_t* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p), 0, bytes, 0x00020000);
}
template <bool CACHED>
__device__ __forceinline__ u32x4 load_row_16(__amdgpu_buffer_rsrc_t rows, int at) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, at, 0, CACHED ? 0 : NT));
}
__device__ __forceinline__ void store_row_16(__amdgpu_buffer_rsrc_t rows, int at, u32x4 v) {
    __builtin_amdgcn_raw_buffer_store_b128(v, rows, at, 0, NT);
}
// How a row lies on the lanes: LPR lanes of a wave hold it alone (64 / LPR rows a wave), or WPR waves of 64 lanes share it; a lane
// holds P pieces of 8 elements, piece number lane + LPR * (wave + WPR * p).
template <int LPR_, int WPR_, int P_>
struct Shape {
    static constexpr int LPR = LPR_, WPR = WPR_, P = P_;
    static constexpr int THREADS = WPR > 4 ? 64 * WPR : 256;
    static constexpr int ROWS = THREADS / (LPR * WPR);           // rows of a workgroup
    static_assert(WPR == 1 || LPR == 64, "rows shared by waves take whole waves");
};
}  // namespace row_ops
}  // namespace tyr
