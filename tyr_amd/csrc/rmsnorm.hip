// Root-mean-square norm with the residual's addition, and its gradients (gfx950).
//
//   h = bf16(x + residual)                     (h = x without a residual; h is the stream that goes on to the next layer)
//   y = h * w * rho,   rho = (mean(h^2) + eps)^-1/2
//   out = bf16(y), or e4m3(y / s) with s = max |y| / 448 of the row: the operand and the row scales of the fp8 GEMM.
//
// Gradients, with g = d_out * w and the gradient d_resid that arrives at h from the layers behind:
//   dx = rho g - (rho^3 / d) (sum_i g_i h_i) h + d_resid        (the gradient of x and of the residual alike)
//   dw = sum over rows of d_out h rho
//
// Statistics, maxima and sums are f32; each result is rounded once.  The statistics are those of the rounded h, which is what the
// backward is given.
//
// HBM-bound: 8 bytes an element (bf16 with a residual, and the backward), 7 with e4m3 out.  A row is read once and stays in
// registers between its statistics and its output.
#include "common.hpp"
#include "launch.hpp"
#include <type_traits>

namespace tyr {

namespace rms {
constexpr float E4M3_MAX = 448.0f;
constexpr float TINY = 0x1p-100f;          // rows below it (zero rows among them) take the scale 1: y / s stays finite

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
struct Add { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct Max { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };

// How a row lies on the lanes: LPR lanes of a wave hold it alone (64 / LPR rows a wave), or WPR waves of 64 lanes share it; a lane
// holds P pieces of 8 elements, piece number lane + LPR * (wave + WPR * p).
template <int LPR_, int WPR_, int P_>
struct Shape {
    static constexpr int LPR = LPR_, WPR = WPR_, P = P_;
    static constexpr int THREADS = WPR > 4 ? 64 * WPR : 256;
    static constexpr int ROWS = THREADS / (LPR * WPR);           // rows of a workgroup
    static_assert(WPR == 1 || LPR == 64, "rows shared by waves take whole waves");
};
}  // namespace rms

template <class S, bool CACHED, bool RESIDUAL, bool E4M3>
__global__ __launch_bounds__(S::THREADS) void rmsnorm_residual_kernel(
    const uint16_t* __restrict__ x, const uint16_t* __restrict__ res, const uint16_t* __restrict__ weight, void* __restrict__ out,
    uint16_t* __restrict__ out_resid, float* __restrict__ row_scale, size_t rows, int d_model, float eps) {
    using namespace rms;
    constexpr int LPR = S::LPR, WPR = S::WPR, P = S::P;
    __shared__ float2 part[S::ROWS][WPR];
    const int lane = threadIdx.x % LPR, wave = threadIdx.x / 64, wr = wave % WPR;
    const int slot = WPR > 1 ? wave / WPR : threadIdx.x / LPR;      // row of the workgroup
    const size_t row = (size_t)blockIdx.x * S::ROWS + slot;
    const int pieces = row < rows ? d_model / 8 : 0;
    const size_t at = row * d_model;
    u32x4 a[P], b[P], w[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int pc = lane + LPR * (wr + WPR * p);
        if (pc < pieces) {
            a[p] = ld_stream_16<CACHED>(x + at + pc * 8);
            if constexpr (RESIDUAL) b[p] = ld_stream_16<CACHED>(res + at + pc * 8);
            w[p] = ld_global_16(weight + pc * 8);
        }
    }
    float h[P][8], sq = 0.0f, top = 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int pc = lane + LPR * (wr + WPR * p);
        if (pc >= pieces) continue;
        unpack8(a[p], h[p]);
        if constexpr (RESIDUAL) {
            float f[8];
            unpack8(b[p], f);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] += h[p][i];
            const u32x4 r16 = pack8(f);
            st_global_16_nt(out_resid + at + pc * 8, r16);
            unpack8(r16, h[p]);
        }
        float wf[8];
        unpack8(w[p], wf);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sq += h[p][i] * h[p][i];
            h[p][i] *= wf[i];
            if constexpr (E4M3) top = fmaxf(top, fabsf(h[p][i]));
        }
    }
    sq = over_lanes<LPR>(sq, Add{});
    if constexpr (E4M3) top = over_lanes<LPR>(top, Max{});
    if constexpr (WPR > 1) {
        if (lane == 0) part[slot][wr] = float2{sq, top};
        __syncthreads();
        sq = 0.0f;
#pragma unroll
        for (int i = 0; i < WPR; ++i) {
            sq += part[slot][i].x;
            if constexpr (E4M3) top = fmaxf(top, part[slot][i].y);
        }
    }
    const float rho = rsqrtf(sq / (float)d_model + eps);
    if constexpr (E4M3) {
        top *= rho;                                                 // max |y|: rho is positive
        const float s = top < TINY ? 1.0f : top / E4M3_MAX, f = rho / s;
        if (lane == 0 && wr == 0 && pieces) row_scale[row] = s;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int pc = lane + LPR * (wr + WPR * p);
            if (pc < pieces)
                st_global_8(static_cast<uint8_t*>(out) + at + pc * 8,
                            u32x2{pack_e4m3(f32x4{h[p][0], h[p][1], h[p][2], h[p][3]} * f), pack_e4m3(f32x4{h[p][4], h[p][5], h[p][6], h[p][7]} * f)});
        }
    } else {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int pc = lane + LPR * (wr + WPR * p);
            if (pc >= pieces) continue;
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = h[p][i] * rho;
            st_global_16_nt(static_cast<uint16_t*>(out) + at + pc * 8, pack8(o));
        }
    }
}

// Gradients.  Workgroup i takes the row groups i, i + gridDim.x, ... and keeps dw of its rows in registers; rows that share a
// workgroup are added through LDS at its end, and it writes one row of part [gridDim.x][d_model].
template <class S, bool CACHED, bool RESID>
__global__ __launch_bounds__(S::THREADS) void rmsnorm_residual_bwd_kernel(
    const uint16_t* __restrict__ d_out, const uint16_t* __restrict__ d_resid, const uint16_t* __restrict__ resid,
    const uint16_t* __restrict__ weight, uint16_t* __restrict__ dx, float* __restrict__ dw_part, size_t rows, int d_model, float eps) {
    using namespace rms;
    constexpr int LPR = S::LPR, WPR = S::WPR, P = S::P;
    __shared__ float2 part[2][S::ROWS][WPR];
    extern __shared__ __attribute__((aligned(16))) float sums[];   // [ROWS][d_model], where a workgroup holds several rows
    const int lane = threadIdx.x % LPR, wave = threadIdx.x / 64, wr = wave % WPR;
    const int slot = WPR > 1 ? wave / WPR : threadIdx.x / LPR;
    const int all = d_model / 8;
    float w[P][8], dw[P][8];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int pc = lane + LPR * (wr + WPR * p);
        u32x4 v = {0, 0, 0, 0};
        if (pc < all) v = ld_global_16(weight + pc * 8);
        unpack8(v, w[p]);
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[p][i] = 0.0f;
    }
    int turn = 0;
    for (size_t first = (size_t)blockIdx.x * S::ROWS; first < rows; first += (size_t)gridDim.x * S::ROWS, turn ^= 1) {
        const size_t row = first + slot;
        const int pieces = row < rows ? all : 0;
        const size_t at = row * d_model;
        u32x4 g16[P], h16[P], r16[P];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int pc = lane + LPR * (wr + WPR * p);
            g16[p] = h16[p] = r16[p] = u32x4{0, 0, 0, 0};
            if (pc < pieces) {
                g16[p] = ld_stream_16<CACHED>(d_out + at + pc * 8);
                h16[p] = ld_stream_16<CACHED>(resid + at + pc * 8);
                if constexpr (RESID) r16[p] = ld_stream_16<CACHED>(d_resid + at + pc * 8);
            }
        }
        float sq = 0.0f, gh = 0.0f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float g[8], h[8];
            unpack8(g16[p], g);
            unpack8(h16[p], h);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sq += h[i] * h[i];
                gh += g[i] * w[p][i] * h[i];
            }
        }
        sq = over_lanes<LPR>(sq, Add{});
        gh = over_lanes<LPR>(gh, Add{});
        if constexpr (WPR > 1) {
            // two sets of sums in turn: a wave that is already at the next row writes the other one
            if (lane == 0) part[turn][slot][wr] = float2{sq, gh};
            __syncthreads();
            sq = gh = 0.0f;
#pragma unroll
            for (int i = 0; i < WPR; ++i) { sq += part[turn][slot][i].x; gh += part[turn][slot][i].y; }
        }
        const float rho = rsqrtf(sq / (float)d_model + eps);
        const float c = rho * rho * rho * (gh / (float)d_model);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int pc = lane + LPR * (wr + WPR * p);
            if (pc >= pieces) continue;
            float g[8], h[8], r[8], o[8];
            unpack8(g16[p], g);
            unpack8(h16[p], h);
            if constexpr (RESID) unpack8(r16[p], r);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                o[i] = rho * (g[i] * w[p][i]) - c * h[i];
                if constexpr (RESID) o[i] += r[i];
                dw[p][i] += g[i] * (h[i] * rho);
            }
            st_global_16_nt(dx + at + pc * 8, pack8(o));
        }
    }
    float* to = dw_part + (size_t)blockIdx.x * d_model;
    if constexpr (S::ROWS > 1) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int pc = lane + LPR * (wr + WPR * p);
            if (pc < all) {
                f32x4* s = reinterpret_cast<f32x4*>(sums + (size_t)slot * d_model + pc * 8);
                s[0] = f32x4{dw[p][0], dw[p][1], dw[p][2], dw[p][3]};
                s[1] = f32x4{dw[p][4], dw[p][5], dw[p][6], dw[p][7]};
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < d_model / 4; i += S::THREADS) {
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < S::ROWS; ++r) v += *reinterpret_cast<const f32x4*>(sums + (size_t)r * d_model + 4 * i);
            *reinterpret_cast<f32x4*>(to + 4 * i) = v;
        }
    } else {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int pc = lane + LPR * (wr + WPR * p);
            if (pc < all) {
                f32x4* s = reinterpret_cast<f32x4*>(to + pc * 8);
                s[0] = f32x4{dw[p][0], dw[p][1], dw[p][2], dw[p][3]};
                s[1] = f32x4{dw[p][4], dw[p][5], dw[p][6], dw[p][7]};
            }
        }
    }
}

// dw = sum of the parts: 8 threads of 4 columns, 32 parts at once, joined through LDS.
__global__ __launch_bounds__(256) void rmsnorm_dweight_kernel(const float* __restrict__ part, uint16_t* __restrict__ dw, int parts, int d_model) {
    __shared__ f32x4 sums[32][8];
    const int c = threadIdx.x % 8, g = threadIdx.x / 8;
    const int col = blockIdx.x * 32 + c * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (col < d_model) {
#pragma unroll 8
        for (int i = g; i < parts; i += 32) v += *reinterpret_cast<const f32x4*>(part + (size_t)i * d_model + col);
    }
    sums[g][c] = v;
    __syncthreads();
    if (g == 0 && col < d_model) {
        for (int i = 1; i < 32; ++i) v += sums[i][c];
        st_global_8(dw + col, u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])});
    }
}

// ------------------------------------------------------------------------------------------
namespace {
template <class F>
void with_shape(int d_model, F go) {
    using namespace rms;
    if (d_model <= 64) go(Shape<8, 1, 1>{});
    else if (d_model <= 128) go(Shape<16, 1, 1>{});
    else if (d_model <= 256) go(Shape<32, 1, 1>{});
    else if (d_model <= 512) go(Shape<64, 1, 1>{});
    else if (d_model <= 1024) go(Shape<64, 1, 2>{});
    else if (d_model <= 2048) go(Shape<64, 2, 2>{});
    else if (d_model <= 4096) go(Shape<64, 4, 2>{});
    else if (d_model <= 8192) go(Shape<64, 8, 2>{});
    else go(Shape<64, 16, 2>{});
}

// workgroups of a backward: parts of dw
template <class S>
size_t bwd_parts(size_t rows) {
    const size_t groups = (rows + S::ROWS - 1) / S::ROWS;
    return groups < 1024 ? groups : 1024;
}
}  // namespace

int launch_rmsnorm_residual(const void* x, const void* residual, const void* weight, void* out, void* out_resid, float* row_scale,
                            size_t rows, int d_model, float eps, int e4m3, hipStream_t stream) {
    const size_t bytes = rows * d_model * ((residual ? 6 : 2) + (e4m3 ? 1 : 2));
    with_shape(d_model, [&](auto shape) {
        using S = decltype(shape);
        auto go = [&](auto cached, auto with_res, auto fp8) {
            launch_kernel((rmsnorm_residual_kernel<S, cached(), with_res(), fp8()>), dim3((unsigned)((rows + S::ROWS - 1) / S::ROWS)),
                          dim3(S::THREADS), 0, stream, static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(residual),
                          static_cast<const uint16_t*>(weight), out, static_cast<uint16_t*>(out_resid), row_scale, rows, d_model, eps);
        };
        auto pick = [&](auto cached) {
            if (residual) { if (e4m3) go(cached, std::true_type{}, std::true_type{}); else go(cached, std::true_type{}, std::false_type{}); }
            else { if (e4m3) go(cached, std::false_type{}, std::true_type{}); else go(cached, std::false_type{}, std::false_type{}); }
        };
        if (bytes <= kStreamCached) pick(std::true_type{}); else pick(std::false_type{});
    });
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

size_t rmsnorm_residual_bwd_workspace_bytes(size_t rows, int d_model) {
    size_t parts = 0;
    with_shape(d_model, [&](auto shape) { parts = bwd_parts<decltype(shape)>(rows); });
    return parts * d_model * sizeof(float);
}

int launch_rmsnorm_residual_bwd(const void* d_out, const void* d_resid, const void* resid, const void* weight, void* dx, void* dweight,
                                size_t rows, int d_model, float eps, void* workspace, hipStream_t stream) {
    const bool cached = rows * d_model * (d_resid ? 8 : 6) <= kStreamCached;
    size_t parts = 0;
    with_shape(d_model, [&](auto shape) {
        using S = decltype(shape);
        parts = bwd_parts<S>(rows);
        const size_t lds = S::ROWS > 1 ? (size_t)S::ROWS * d_model * sizeof(float) : 0;
        auto go = [&](auto in_cache, auto with_resid) {
            launch_kernel((rmsnorm_residual_bwd_kernel<S, in_cache(), with_resid()>), dim3((unsigned)parts), dim3(S::THREADS), lds, stream,
                          static_cast<const uint16_t*>(d_out), static_cast<const uint16_t*>(d_resid), static_cast<const uint16_t*>(resid),
                          static_cast<const uint16_t*>(weight), static_cast<uint16_t*>(dx), static_cast<float*>(workspace), rows, d_model, eps);
        };
        if (d_resid) { if (cached) go(std::true_type{}, std::true_type{}); else go(std::false_type{}, std::true_type{}); }
        else { if (cached) go(std::true_type{}, std::false_type{}); else go(std::false_type{}, std::false_type{}); }
    });
    if (hipGetLastError() != hipSuccess) return -1;
    launch_kernel(rmsnorm_dweight_kernel, dim3((unsigned)((d_model + 31) / 32)), dim3(256), 0, stream, static_cast<const float*>(workspace),
                  static_cast<uint16_t*>(dweight), (int)parts, d_model);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tyr
