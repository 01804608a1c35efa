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
// registers between its statistics and its output.  Stores go past the caches (plain ones: 65536 x 1024 91.5 us, 87 so; 35552 x 128 4.5, 3.8).
#include "common.hpp"
#include "launch.hpp"
#include <type_traits>
#include <utility>

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
    each<P>([&](auto p) {
        const int pc = lane + LPR * (wr + WPR * p);
        if (pc < pieces) {
            a[p] = ld_stream_16<CACHED>(x + at + pc * 8);
            if constexpr (RESIDUAL) b[p] = ld_stream_16<CACHED>(res + at + pc * 8);
            w[p] = ld_global_16(weight + pc * 8);
            __builtin_amdgcn_sched_barrier(0);                      // all are asked for before one is waited for
        }
    });
    float h[P][8], sq = 0.0f, top = 0.0f;
    each<P>([&](auto p) {
        const int pc = lane + LPR * (wr + WPR * p);
        if (pc >= pieces) return;
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
    });
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
    const float mean = sq / (float)d_model + eps;
    float rho = rsqrtf(mean);
    if (__builtin_expect(any_beyond<LPR>(mean), 0) && beyond(mean)) {
        auto element = [&](int pc, float (&f)[8]) {
            unpack8(ld_global_16(x + at + pc * 8), f);
            if constexpr (RESIDUAL) {
                float r[8];
                unpack8(ld_global_16(res + at + pc * 8), r);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] += r[i];
                unpack8(pack8(f), f);
            }
        };
        float f[8], wf[8], most = sqrtf(eps);
        for (int pc = lane; pc < pieces; pc += LPR) {
            element(pc, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(f[i]));
        }
        const float k = power_for(over_lanes<LPR>(most, Max{}));
        sq = top = 0.0f;
        for (int pc = lane; pc < pieces; pc += LPR) {
            element(pc, f);
            unpack8(ld_global_16(weight + pc * 8), wf);
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] *= k;
                s += f[i] * f[i];
                top = fmaxf(top, fabsf(f[i] * wf[i]));
            }
            sq += s;
        }
        sq = over_lanes<LPR>(sq, Add{});
        top = over_lanes<LPR>(top, Max{});
        rho = rsqrtf(sq / (float)d_model + eps * k * k);
        each<P>([&](auto p) {
            const int pc = lane + LPR * (wr + WPR * p);
            if (pc >= pieces) return;
            element(pc, h[p]);
            unpack8(ld_global_16(weight + pc * 8), wf);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[p][i] = h[p][i] * k * wf[i];
        });
    }
    if constexpr (E4M3) {
        top *= rho;                                                 // max |y|: rho is positive
        const float s = top < TINY ? 1.0f : top / E4M3_MAX, f = rho / s;
        if (lane == 0 && wr == 0 && pieces) row_scale[row] = s;
        each<P>([&](auto p) {
            const int pc = lane + LPR * (wr + WPR * p);
            if (pc < pieces)
                st_global_8(static_cast<uint8_t*>(out) + at + pc * 8,
                            u32x2{pack_e4m3(f32x4{h[p][0], h[p][1], h[p][2], h[p][3]} * f), pack_e4m3(f32x4{h[p][4], h[p][5], h[p][6], h[p][7]} * f)});
        });
    } else {
        each<P>([&](auto p) {
            const int pc = lane + LPR * (wr + WPR * p);
            if (pc >= pieces) return;
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = h[p][i] * rho;
            st_global_16_nt(static_cast<uint16_t*>(out) + at + pc * 8, pack8(o));
        });
    }
}

// Gradients.  Workgroups of 16 waves (or as many of them as whole rows need): as many row slots as fit, slot s of workgroup i takes the rows ROWS (i + k gridDim.x) + s, the
// next one's loads under way while it works on one, and keeps dw of its rows in registers.  The slots are added through LDS at the
// end, half of them to the other half at a time, and the workgroup writes one row of part [gridDim.x][d_model].
// 65536 x 1024 85 us of reading and writing 537 MB and 5 us for the parts; 2000 x 4096 12.5 and 3.  (1024 workgroups of four waves: 91 and
// 14, and 17 MB of parts; two pieces a lane, spilling: 93 and 15; 512 workgroups: 86 and 15.)
template <class S, bool CACHED, bool RESID>
__global__ __launch_bounds__(1024) void rmsnorm_residual_bwd_kernel(
    const uint16_t* __restrict__ d_out, const uint16_t* __restrict__ d_resid, const uint16_t* __restrict__ resid,
    const uint16_t* __restrict__ weight, uint16_t* __restrict__ dx, float* __restrict__ dw_part, uint16_t* __restrict__ dw_out, size_t rows, int d_model, float eps) {
    using namespace rms;
    constexpr int LPR = S::LPR, WPR = S::WPR, P = S::P, ROWS = 1024 / (LPR * WPR);
    __shared__ float2 part[2][ROWS][WPR];
    extern __shared__ __attribute__((aligned(16))) float sums[];   // [ROWS / 2][d_model]
    const int lane = threadIdx.x % LPR, wave = threadIdx.x / 64, wr = wave % WPR;
    const int slot = WPR > 1 ? wave / WPR : threadIdx.x / LPR;
    int pc[P], at[P];                                            // this lane's elements of a row; their place in a group of rows
    bool has[P];
    constexpr bool TIGHT = P > 1;                                // registers for the rows as they came only
    float w[P][8], dw[P][8];
    u32x4 w16[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        pc[p] = 8 * (lane + LPR * (wr + WPR * p));
        has[p] = pc[p] < d_model;
        at[p] = has[p] ? 2 * (slot * d_model + pc[p]) : NOWHERE;
        w16[p] = has[p] ? ld_global_16(weight + pc[p]) : u32x4{0, 0, 0, 0};
        unpack8(w16[p], w[p]);
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[p][i] = 0.0f;
    }
    // A group of ROWS rows is a buffer: what lies behind the last row is read as 0 and not written.
    struct Row { u32x4 g[P], h[P], r[P]; };
    auto group = [&](const uint16_t* x, size_t first) {
        const size_t n = first < rows ? (rows - first < (size_t)ROWS ? rows - first : (size_t)ROWS) : 0;
        return rows_rsrc(x + first * d_model, (int)n * d_model * 2);
    };
    auto read = [&](Row& o, size_t first) {
        const auto g = group(d_out, first), h = group(resid, first), r = group(RESID ? d_resid : resid, first);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            o.h[p] = load_row_16<CACHED>(h, at[p]);
            o.g[p] = load_row_16<CACHED>(g, at[p]);
            if constexpr (RESID) o.r[p] = load_row_16<CACHED>(r, at[p]);
        }
    };
    int turn = 0;
    // unpacks a second time what is to be kept in its 16 bits between
    auto again = [](u32x4 v, float (&f)[8]) {
        asm volatile("" : "+v"(v));
        unpack8(v, f);
    };
    auto work = [&](Row& o, size_t first) {
        float sq = 0.0f, gwh = 0.0f, g[P][8], h[P][8], gh[P][8];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            unpack8(o.g[p], g[p]);
            unpack8(o.h[p], h[p]);
            if constexpr (TIGHT) again(w16[p], w[p]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sq += h[p][i] * h[p][i];
                gh[p][i] = g[p][i] * h[p][i];
                gwh += gh[p][i] * w[p][i];
            }
        }
        sq = over_lanes<LPR>(sq, Add{});
        gwh = over_lanes<LPR>(gwh, Add{});
        if constexpr (WPR > 1) {
            // two sets of sums in turn: a wave that is already at the next row writes the other one
            if (lane == 0) part[turn][slot][wr] = float2{sq, gwh};
            __syncthreads();
            sq = gwh = 0.0f;
#pragma unroll
            for (int i = 0; i < WPR; ++i) { sq += part[turn][slot][i].x; gwh += part[turn][slot][i].y; }
            turn ^= 1;
        }
        const bool real = first + slot < rows;
        const float mean = sq / (float)d_model + eps;
        float rho = real ? rsqrtf(mean) : 0.0f;
        float c = gwh / (float)d_model * rho * rho * rho;            // in this order: rho^3 alone leaves f32 for rows of 1e13 or 1e-13
        float rho_x = rho;                                           // of dx; the other is that of h as it stands in o
        if (__builtin_expect(any_beyond<LPR>(mean), 0) && real && beyond(mean)) {
            const uint16_t *hr = resid + (first + slot) * d_model, *gr = d_out + (first + slot) * d_model;
            float f[8], e[8], wf[8], most = sqrtf(eps);
            for (int i0 = 8 * lane; i0 < d_model; i0 += 8 * LPR) {
                unpack8(ld_global_16(hr + i0), f);
#pragma unroll
                for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(f[i]));
            }
            const float k = power_for(over_lanes<LPR>(most, Max{}));
            sq = gwh = 0.0f;
            for (int i0 = 8 * lane; i0 < d_model; i0 += 8 * LPR) {
                unpack8(ld_global_16(hr + i0), f);
                unpack8(ld_global_16(gr + i0), e);
                unpack8(ld_global_16(weight + i0), wf);
                float s = 0.0f, t = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    f[i] *= k;
                    s += f[i] * f[i];
                    t += e[i] * f[i] * wf[i];
                }
                sq += s;
                gwh += t;
            }
            sq = over_lanes<LPR>(sq, Add{});
            gwh = over_lanes<LPR>(gwh, Add{});
            rho = rsqrtf(sq / (float)d_model + eps * k * k);
            c = gwh / (float)d_model * rho * rho * rho * k;
            rho_x = rho * k;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                unpack8(o.h[p], h[p]);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    h[p][i] *= k;                                    // what underflows is nothing beside the row's largest
                    gh[p][i] = g[p][i] * h[p][i];
                }
                o.h[p] = pack8(h[p]);
            }
        }
        const auto to = group(dx, first);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float r[8], o8[8];
            if constexpr (RESID) unpack8(o.r[p], r);
            if constexpr (TIGHT) {
                again(o.g[p], g[p]);
                again(o.h[p], h[p]);
                again(w16[p], w[p]);
#pragma unroll
                for (int i = 0; i < 8; ++i) gh[p][i] = g[p][i] * h[p][i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float gw = g[p][i] * w[p][i];
                o8[i] = fmaf(-c, h[p][i], RESID ? fmaf(rho_x, gw, r[i]) : rho_x * gw);
                dw[p][i] = fmaf(gh[p][i], rho, dw[p][i]);
            }
            store_row_16(to, at[p], pack8(o8));
        }
    };
    const size_t stride = (size_t)gridDim.x * ROWS;
    Row now, next;
    read(now, (size_t)blockIdx.x * ROWS);
    for (size_t first = (size_t)blockIdx.x * ROWS; first < rows; first += stride) {      // the same for all slots: they meet at barriers
        read(next, first + stride);
        work(now, first);
        now = next;
    }
#pragma unroll
    for (int n = ROWS; n > 1; n = (n + 1) / 2) {
        const int half = (n + 1) / 2;
        __syncthreads();
        if (slot >= half && slot < n)
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (has[p]) {
                    f32x4* s = reinterpret_cast<f32x4*>(sums + (size_t)(slot - half) * d_model + pc[p]);
                    s[0] = f32x4{dw[p][0], dw[p][1], dw[p][2], dw[p][3]};
                    s[1] = f32x4{dw[p][4], dw[p][5], dw[p][6], dw[p][7]};
                }
        __syncthreads();
        if (slot < n - half)
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (has[p]) {
                    const f32x4* s = reinterpret_cast<const f32x4*>(sums + (size_t)slot * d_model + pc[p]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) dw[p][i] += s[i / 4][i % 4];
                }
    }
    if (slot == 0)
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (has[p] && dw_out) st_global_16(dw_out + pc[p], pack8(dw[p]));      // the only workgroup
            else if (has[p]) {
                f32x4* s = reinterpret_cast<f32x4*>(dw_part + (size_t)blockIdx.x * d_model + pc[p]);
                s[0] = f32x4{dw[p][0], dw[p][1], dw[p][2], dw[p][3]};
                s[1] = f32x4{dw[p][4], dw[p][5], dw[p][6], dw[p][7]};
            }
}

// dw = sum of the parts: 8 threads of 4 columns, 32 parts at once, joined through LDS.  It is all latency (1024 threads for 128
// parts at once take as long).
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
#pragma unroll
        for (int i = 1; i < 32; ++i) v += sums[i][c];
        st_global_8(dw + col, u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])});
    }
}

// ------------------------------------------------------------------------------------------
namespace {
// Of the backward: one piece a lane, whose values, weights and sums fill the registers, as long as 16 waves hold a row so.  Of waves without
// work there are fewer with five to a row (22880 x 2080 87 us with eight, 69 so; 1000 x 2560 10.1, 10.5) and ten, two workgroups a CU.
template <class F>
void with_bwd_shape(int d_model, F go) {
    using namespace rms;
    if (d_model <= 64) go(Shape<8, 1, 1>{});
    else if (d_model <= 128) go(Shape<16, 1, 1>{});
    else if (d_model <= 256) go(Shape<32, 1, 1>{});
    else if (d_model <= 512) go(Shape<64, 1, 1>{});
    else if (d_model <= 1024) go(Shape<64, 2, 1>{});
    else if (d_model <= 2048) go(Shape<64, 4, 1>{});
    else if (d_model <= 2560) go(Shape<64, 5, 1>{});
    else if (d_model <= 4096) go(Shape<64, 8, 1>{});
    else if (d_model <= 5120) go(Shape<64, 10, 1>{});
    else if (d_model <= 8192) go(Shape<64, 16, 1>{});
    else go(Shape<64, 16, 2>{});
}
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

// Rows of so many groups at most are one workgroup's, which then has dw: 2 rows of 2048 5.7 us by two launches, 3.3 so; two groups 5.9, 4.5;
// three 5.7, 6.7.
constexpr size_t ALONE = 2;
// workgroups of a backward: parts of dw.  One a CU; of ten waves two, where the rows outweigh the parts (5700 x 4400 51.7 us with one, 47.5 so;
// 2000 x 5120 20.0, 21.2).
template <class S>
size_t bwd_parts(size_t rows) {
    constexpr int ROWS = 1024 / (S::LPR * S::WPR);
    const size_t groups = (rows + ROWS - 1) / ROWS, most = groups <= ALONE ? 1 : S::WPR == 10 && rows >= 4096 ? 512 : 256;
    return groups < most ? groups : most;
}
}  // namespace

bool rmsnorm_residual_fits(size_t rows, int d_model) {
    bool fits = false;
    with_shape(d_model, [&](auto shape) {
        using S = decltype(shape);
        fits = (rows + S::ROWS - 1) / S::ROWS * S::THREADS < ((size_t)1 << 32);
    });
    return fits;
}

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
    with_bwd_shape(d_model, [&](auto shape) { parts = bwd_parts<decltype(shape)>(rows); });
    return parts * d_model * sizeof(float);
}

int launch_rmsnorm_residual_bwd(const void* d_out, const void* d_resid, const void* resid, const void* weight, void* dx, void* dweight,
                                size_t rows, int d_model, float eps, void* workspace, hipStream_t stream) {
    const bool cached = rows * d_model * (d_resid ? 8 : 6) <= kStreamCached;
    size_t parts = 0;
    with_bwd_shape(d_model, [&](auto shape) {
        using S = decltype(shape);
        parts = bwd_parts<S>(rows);
        constexpr int ROWS = 1024 / (S::LPR * S::WPR);
        const size_t lds = (size_t)(ROWS / 2) * d_model * sizeof(float);        // at most 16 KB
        auto go = [&](auto in_cache, auto with_resid) {
            launch_kernel((rmsnorm_residual_bwd_kernel<S, in_cache(), with_resid()>), dim3((unsigned)parts), dim3(S::LPR * S::WPR * ROWS), lds, stream,
                          static_cast<const uint16_t*>(d_out), static_cast<const uint16_t*>(d_resid), static_cast<const uint16_t*>(resid),
                          static_cast<const uint16_t*>(weight), static_cast<uint16_t*>(dx), static_cast<float*>(workspace),
                          parts == 1 ? static_cast<uint16_t*>(dweight) : nullptr, rows, d_model, eps);
        };
        if (d_resid) { if (cached) go(std::true_type{}, std::true_type{}); else go(std::false_type{}, std::true_type{}); }
        else { if (cached) go(std::true_type{}, std::false_type{}); else go(std::false_type{}, std::false_type{}); }
    });
    if (hipGetLastError() != hipSuccess) return -1;
    if (parts == 1) return 0;
    launch_kernel(rmsnorm_dweight_kernel, dim3((unsigned)((d_model + 31) / 32)), dim3(256), 0, stream, static_cast<const float*>(workspace),
                  static_cast<uint16_t*>(dweight), (int)parts, d_model);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tyr
