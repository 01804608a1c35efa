// Layer norm with the residual's addition (or without), and its gradients (gfx950).
//
//   h = bf16(x + residual)                     (h = x without a residual; h is the stream that goes on to the next layer)
//   n = (h - mean) rho,   rho = (var + eps)^-1/2, mean and var of the row
//   out = bf16(n w + bias)                     (without a bias: n w)
//
// Gradients, with g = d_out w and the gradient d_resid that arrives at h from the layers behind:
//   dx = rho (g - mean(g) - n mean(g n)) + d_resid              (the gradient of x and of the residual alike)
//   dw = sum over rows of d_out n,   dbias = sum over rows of d_out
//
// Reference semantics of the form with a residual and a bias: Tyr/GPU/Kernels/FusedLayerNorm.lean:28-140
// (tkFusedLayerNormResidual1024), expected values Examples/GPU/RunLayerNorm.lean:27-33.
//
// Statistics and sums are f32, each result is rounded once.  The variance is that of the differences from the mean: of each wave's elements
// about their own mean, then of the row's waves together.  Rows that f32 does not hold the squares of are scaled by a power of two.
//
// HBM-bound: 8 bytes an element with a residual, 4 without, 8 (6 without d_resid) in the backward.  A row is read once and stays in registers.
#include "launch.hpp"
#include "rows.hpp"

namespace tyr {

// WPR waves per row; a lane holds P <= 2 pieces (8 bf16) of it, lane, lane + LPR * WPR, so that all loads of a row, weights
// included, are under way at once and many waves share the chip (one wave per row, up to 16 pieces a lane: 2222 x 4096
// 16.8 us, 300 x 8192 17; so 13.1 and 7.1).  65536 x 1024 without a residual 43.8 us, 6.1 TB/s.
template <class S, bool CACHED, bool RESIDUAL, bool BIAS>
__global__ __launch_bounds__(S::THREADS) void layernorm_residual_kernel(
    const uint16_t* __restrict__ x, const uint16_t* __restrict__ res, const uint16_t* __restrict__ weight,
    const uint16_t* __restrict__ bias, uint16_t* __restrict__ out, uint16_t* __restrict__ out_resid, size_t rows,
    int d_model, float eps, bool in_place) {
    using namespace row_ops;
    constexpr int LPR = S::LPR, WPR = S::WPR, P = S::P;
    __shared__ float2 part[S::ROWS][WPR];
    const int lane = threadIdx.x % LPR, wave = threadIdx.x / 64, wr = wave % WPR;
    const int slot = WPR > 1 ? wave / WPR : threadIdx.x / LPR;      // row of the workgroup
    const size_t row = (size_t)blockIdx.x * S::ROWS + slot;
    const int pieces = row < rows ? d_model / 8 : 0;
    const size_t at = row * d_model;
    float v[P][8];
    u32x4 a[P], b[P], w[P], bi[P];
    each<P>([&](auto p) {
        const int pc = lane + LPR * (wr + WPR * p);
        if (pc < pieces) {
            a[p] = ld_stream_16<CACHED>(x + at + pc * 8);
            if constexpr (RESIDUAL) b[p] = ld_stream_16<CACHED>(res + at + pc * 8);
            w[p] = ld_global_16(weight + pc * 8);
            if constexpr (BIAS) bi[p] = ld_global_16(bias + pc * 8);
            __builtin_amdgcn_sched_barrier(0);                      // all are asked for before one is waited for
        }
    });
    float sum = 0.0f;
    each<P>([&](auto p) {
        const int pc = lane + LPR * (wr + WPR * p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[p][i] = 0.0f;
        if (pc >= pieces) return;
        unpack8(a[p], v[p]);
        if constexpr (RESIDUAL) {
            float f[8];
            unpack8(b[p], f);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = v[p][i] + f[i];
            const u32x4 r16 = pack8(f);                             // out_resid is the bf16-rounded sum ...
            st_global_16_nt(out_resid + at + pc * 8, r16);
            unpack8(r16, v[p]);                                     // ... and the statistics are taken from it
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += v[p][i];
    });
    // mean and sum of squares about it: of each wave's elements, then of the row's waves together
    auto elements = [](int i, int pieces) {                         // of wave i of a row
        int c = 0;
#pragma unroll
        for (int p = 0; p < P; ++p) c += max(0, min(LPR, pieces - LPR * (i + WPR * p)));
        return 8.0f * (float)c;
    };
    float mean = over_lanes<LPR>(sum, Add{}) / fmaxf(elements(wr, pieces), 1.0f);
    float sq = 0.0f;
    each<P>([&](auto p) {
        if (lane + LPR * (wr + WPR * p) < pieces) {
#pragma unroll
            for (int i = 0; i < 8; ++i) { const float c = v[p][i] - mean; sq += c * c; }
        }
    });
    sq = over_lanes<LPR>(sq, Add{});
    if constexpr (WPR > 1) {
        if (lane == 0) part[slot][wr] = float2{mean, sq};
        __syncthreads();
    }
    auto joined = [&](int slot, int pieces) {                       // mean and sum of squares of a row
        float2 q[WPR];
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < WPR; ++i) {
            q[i] = part[slot][i];
            total += q[i].x * elements(i, pieces);
        }
        const float mean = total / (float)d_model;
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < WPR; ++i) { const float d = q[i].x - mean; sq += q[i].y + elements(i, pieces) * d * d; }
        return float2{mean, sq};
    };
    if constexpr (WPR > 1) {
        const float2 of = joined(slot, pieces);
        mean = of.x;
        sq = of.y;
    }
    float var = sq / (float)d_model + eps;
    // A row that is scaled is read again: h from out_resid, as x and residual may be what has been written, and without a residual x, which out may
    // be (in_place; the compiler takes them for different).  There the row's waves wait for each other before they write, at a barrier, which is
    // all waves' of the workgroup: each looks at all of its rows, in the same steps.  (At every call: 32768 x 1536 37.6 us instead of 36.4.)
    constexpr bool MAY_WAIT = WPR > 1 && !RESIDUAL;
    bool waits = false;
    if (MAY_WAIT && in_place) {
#pragma unroll
        for (int s = 0; s < S::ROWS; ++s) {
            const float2 of = joined(s, row - slot + s < rows ? d_model / 8 : 0);
            const float v = of.y / (float)d_model + eps;
            waits |= beyond(v);
            if (s == slot) {
                mean = of.x;
                var = v;
            }
        }
        waits = __builtin_amdgcn_readfirstlane(waits);
    }
    float inv_std = rsqrtf(var);
    if (__builtin_expect(any_beyond<LPR>(var), 0) && beyond(var)) {
        if constexpr (RESIDUAL) __threadfence_block();              // other lanes wrote it
        const uint16_t* const h = RESIDUAL ? out_resid : x;
        auto element = [&](int pc, float (&f)[8]) { unpack8(ld_global_16(h + at + pc * 8), f); };
        float f[8], most = sqrtf(eps);
        for (int pc = lane; pc < pieces; pc += LPR) {
            element(pc, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(f[i]));
        }
        const float k = power_for(over_lanes<LPR>(most, Max{}));
        sum = 0.0f;
        for (int pc = lane; pc < pieces; pc += LPR) {
            element(pc, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += f[i] * k;
        }
        mean = over_lanes<LPR>(sum, Add{}) / (float)d_model;
        sq = 0.0f;
        for (int pc = lane; pc < pieces; pc += LPR) {
            element(pc, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) { const float c = f[i] * k - mean; sq += c * c; }
        }
        sq = over_lanes<LPR>(sq, Add{});
        const float scaled = sq / (float)d_model + eps * k * k;
        inv_std = scaled < 0x1p-126f && eps > 0.0f ? 1.0f : rsqrtf(scaled);      // equal elements, n = 0: eps k^2 has left f32, eps is not 0
        each<P>([&](auto p) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[p][i] *= k;
        });
    }
    if (MAY_WAIT && __builtin_expect(waits, 0)) __syncthreads();
    each<P>([&](auto p) {
        const int pc = lane + LPR * (wr + WPR * p);
        if (pc >= pieces) return;
        float wf[8], bf[8], o[8];
        unpack8(w[p], wf);
        if constexpr (BIAS) unpack8(bi[p], bf);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float n = (v[p][i] - mean) * inv_std;
            o[i] = BIAS ? n * wf[i] + bf[i] : n * wf[i];
        }
        st_global_16_nt(out + at + pc * 8, pack8(o));
    });
}

// Gradients.  Workgroups of 16 waves (or as many of them as whole rows need): as many row slots as fit, slot s of workgroup i takes the rows
// ROWS (i + k gridDim.x) + s, the next one's loads under way while it works on one, and keeps dw and dbias of its rows in registers.  The slots
// are added through LDS at the end, half of them to the other half at a time, and the workgroup writes one row of part [gridDim.x][2][d_model].
// 65536 x 1024 with d_resid 89 us (the least of 40 launches 86), 6.0 TB/s, and 5 for the parts; 2000 x 4096 15.1 (13.7) and 3 to 5.  Wide rows are nearly bound by the vector units (a row of
// 5120 takes each of its ten waves some 260 instructions): 20000 x 5120 155 us, 5.3 TB/s.  Two and three rows ahead 2 to 60 % slower (registers).
template <class S, bool CACHED, bool RESID>
__global__ __launch_bounds__(1024) void layernorm_residual_bwd_kernel(
    const uint16_t* __restrict__ d_out, const uint16_t* __restrict__ d_resid, const uint16_t* __restrict__ resid,
    const uint16_t* __restrict__ weight, uint16_t* __restrict__ dx, float* __restrict__ part_out, uint16_t* __restrict__ dw_out,
    uint16_t* __restrict__ db_out, size_t rows, int d_model, float eps) {
    using namespace row_ops;
    constexpr int LPR = S::LPR, WPR = S::WPR, ROWS = 1024 / (LPR * WPR);
    static_assert(S::P == 1, "a lane holds one piece of a row");
    constexpr int JOINED = WPR <= 2 ? 2 : WPR <= 4 ? 4 : WPR <= 8 ? 8 : 16;      // lanes that add the sums of a row's waves, one of them each
    __shared__ f32x4 part[2][ROWS][WPR];
    extern __shared__ __attribute__((aligned(16))) float sums[];   // [ROWS / 2][2][d_model]
    const int lane = threadIdx.x % LPR, wave = threadIdx.x / 64, wr = wave % WPR;
    const int slot = WPR > 1 ? wave / WPR : threadIdx.x / LPR;
    const int pc = 8 * (lane + LPR * wr);                          // this lane's elements of a row
    const bool has = pc < d_model;
    const int at = has ? 2 * (slot * d_model + pc) : NOWHERE;      // their place in a group of rows
    const float inv_d = 1.0f / (float)d_model;
    auto elements = [&](int i) { return 8.0f * (float)max(0, min(LPR, d_model / 8 - LPR * i)); };      // of wave i of a row
    const float n_mine = fmaxf(elements(wr), 1.0f), inv_mine = 1.0f / n_mine;
    // What the rounding of a reciprocal lacks.  With it a sum's quotient is exact where that is a number of f32, as for rows of equal elements, which
    // would have a variance, large beside eps, about a mean that is off by a rounding.  2000 x 4096 19.8 us, 19.6 without.
    const float lacks_d = fmaf(-inv_d, (float)d_model, 1.0f) * inv_d, lacks_mine = fmaf(-inv_mine, n_mine, 1.0f) * inv_mine;
    const int other = lane % JOINED;                               // the wave whose sums this lane reads
    const float others = other < WPR ? elements(other) : 0.0f;
    float w[8], dw[8], db[8];
    unpack8(has ? ld_global_16(weight + pc) : u32x4{0, 0, 0, 0}, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[i] = db[i] = 0.0f;
    // A group of ROWS rows is a buffer: what lies behind the last row is read as 0 and not written.
    struct Row { u32x4 g, h, r; };
    auto group = [&](const uint16_t* x, size_t first) {
        const size_t n = first < rows ? (rows - first < (size_t)ROWS ? rows - first : (size_t)ROWS) : 0;
        return rows_rsrc(x + first * d_model, (int)n * d_model * 2);
    };
    auto read = [&](Row& o, size_t first) {
        o.h = load_row_16<CACHED>(group(resid, first), at);
        o.g = load_row_16<CACHED>(group(d_out, first), at);
        if constexpr (RESID) o.r = load_row_16<CACHED>(group(d_resid, first), at);
    };
    int turn = 0;
    auto work = [&](const Row& o, size_t first) {
        float g[8], h[8], sum = 0.0f;
        unpack8(o.h, h);
        unpack8(o.g, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += h[i];
        // of the wave's elements: their mean, and about it the sums of squares, of g w and of g w times the difference
        sum = over_lanes<LPR>(sum, Add{});
        float mean = fmaf(sum, inv_mine, sum * lacks_mine), sq = 0.0f, gw = 0.0f, gwc = 0.0f;
        const float here = has ? mean : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = h[i] - here, a = g[i] * w[i];
            sq += c * c;
            gw += a;
            gwc += a * c;
        }
        sq = over_lanes<LPR>(sq, Add{});
        gw = over_lanes<LPR>(gw, Add{});
        gwc = over_lanes<LPR>(gwc, Add{});
        if constexpr (WPR > 1) {
            // two sets of sums in turn: a wave that is already at the next row writes the other one
            if (lane == 0) part[turn][slot][wr] = f32x4{mean, sq, gw, gwc};
            __syncthreads();
            if constexpr (WPR == 2) {
                const f32x4 q0 = part[turn][slot][0], q1 = part[turn][slot][1];
                const float n0 = elements(0), n1 = elements(1);
                sum = q0[0] * n0 + q1[0] * n1;
                mean = fmaf(sum, inv_d, sum * lacks_d);
                const float d0 = q0[0] - mean, d1 = q1[0] - mean;
                sq = q0[1] + n0 * d0 * d0 + (q1[1] + n1 * d1 * d1);
                gw = q0[2] + q1[2];
                gwc = q0[3] + q0[2] * d0 + (q1[3] + q1[2] * d1);
            } else {                                                 // a wave's sums a lane, not all of them in every lane: 4096 x 5120 54.9 -> 41.2 us
                const f32x4 q = part[turn][slot][min(other, WPR - 1)];
                const bool real = WPR == JOINED || other < WPR;
                sum = over_lanes<JOINED>(q[0] * others, Add{});
                mean = fmaf(sum, inv_d, sum * lacks_d);
                const float d = q[0] - mean;
                sq = over_lanes<JOINED>(real ? q[1] + others * d * d : 0.0f, Add{});
                gw = over_lanes<JOINED>(real ? q[2] : 0.0f, Add{});
                gwc = over_lanes<JOINED>(real ? q[3] + q[2] * d : 0.0f, Add{});
            }
            turn ^= 1;
        }
        const bool real = first + slot < rows;
        const float var = sq * inv_d + eps;
        float rho = real ? rsqrtf(var) : 0.0f;
        float rho_x = rho;                                           // of dx; the other is that of h as it stands in registers
        float c = gwc * inv_d * rho * rho * rho;                     // in this order: rho^3 alone leaves f32 for rows of 1e13 or 1e-13
        if (__builtin_expect(any_beyond<LPR>(var), 0) && real && beyond(var)) {
            const uint16_t *hr = resid + (first + slot) * d_model, *gr = d_out + (first + slot) * d_model;
            float f[8], e[8], wf[8], most = sqrtf(eps);
            for (int i0 = 8 * lane; i0 < d_model; i0 += 8 * LPR) {
                unpack8(ld_global_16(hr + i0), f);
#pragma unroll
                for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(f[i]));
            }
            const float k = power_for(over_lanes<LPR>(most, Max{}));
            sum = sq = gw = gwc = 0.0f;
            for (int i0 = 8 * lane; i0 < d_model; i0 += 8 * LPR) {
                unpack8(ld_global_16(hr + i0), f);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += f[i] * k;
            }
            mean = over_lanes<LPR>(sum, Add{}) / (float)d_model;
            for (int i0 = 8 * lane; i0 < d_model; i0 += 8 * LPR) {
                unpack8(ld_global_16(hr + i0), f);
                unpack8(ld_global_16(gr + i0), e);
                unpack8(ld_global_16(weight + i0), wf);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float d = f[i] * k - mean, a = e[i] * wf[i];
                    sq += d * d;
                    gw += a;
                    gwc += a * d;
                }
            }
            sq = over_lanes<LPR>(sq, Add{});
            gw = over_lanes<LPR>(gw, Add{});
            gwc = over_lanes<LPR>(gwc, Add{});
            const float scaled = sq / (float)d_model + eps * k * k;
            rho = rsqrtf(scaled);
            rho_x = rho * k;
            if (scaled < 0x1p-126f && eps > 0.0f) {                  // equal elements, n = 0: eps k^2 has left f32, eps is not 0
                rho = 1.0f;
                rho_x = 1.0f / sqrtf(eps);
            }
            c = gwc * inv_d * rho * rho * rho * k;
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] *= k;                   // what underflows is nothing beside the row's largest
        }
        const float m = gw * inv_d * rho_x;
        float r[8], o8[8];
        if constexpr (RESID) unpack8(o.r, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = h[i] - mean, a = fmaf(rho_x, g[i] * w[i], RESID ? r[i] - m : -m);
            o8[i] = fmaf(-c, d, a);
            dw[i] = fmaf(g[i], d * rho, dw[i]);
            db[i] += g[i];
        }
        store_row_16(group(dx, first), at, pack8(o8));
    };
    const size_t stride = (size_t)gridDim.x * ROWS;
    Row now, next;
    read(now, (size_t)blockIdx.x * ROWS);
    for (size_t first = (size_t)blockIdx.x * ROWS; first < rows; first += stride) {      // the same for all slots: they meet at barriers
        read(next, first + stride);
        work(now, first);
        now = next;
    }
    auto place = [&](float* to) {
        f32x4* s = reinterpret_cast<f32x4*>(to + pc);
        s[0] = f32x4{dw[0], dw[1], dw[2], dw[3]};
        s[1] = f32x4{dw[4], dw[5], dw[6], dw[7]};
        s = reinterpret_cast<f32x4*>(to + d_model + pc);
        s[0] = f32x4{db[0], db[1], db[2], db[3]};
        s[1] = f32x4{db[4], db[5], db[6], db[7]};
    };
#pragma unroll
    for (int n = ROWS; n > 1; n = (n + 1) / 2) {
        const int half = (n + 1) / 2;
        __syncthreads();
        if (slot >= half && slot < n && has) place(sums + (size_t)(slot - half) * 2 * d_model);
        __syncthreads();
        if (slot < n - half && has) {
            const f32x4* s = reinterpret_cast<const f32x4*>(sums + (size_t)slot * 2 * d_model + pc);
            const f32x4* t = reinterpret_cast<const f32x4*>(sums + (size_t)slot * 2 * d_model + d_model + pc);
#pragma unroll
            for (int i = 0; i < 8; ++i) { dw[i] += s[i / 4][i % 4]; db[i] += t[i / 4][i % 4]; }
        }
    }
    if (slot == 0 && has) {
        if (dw_out) {                                                // the only workgroup
            st_global_16(dw_out + pc, pack8(dw));
            if (db_out) st_global_16(db_out + pc, pack8(db));
        } else {
            place(part_out + (size_t)blockIdx.x * 2 * d_model);
        }
    }
}

// dw and dbias = sum of the parts: 8 threads of 4 columns, 32 parts at once, joined through LDS.  It is all latency.
__global__ __launch_bounds__(256) void layernorm_dweight_kernel(const float* __restrict__ part, uint16_t* __restrict__ dw, uint16_t* __restrict__ db,
                                                                int parts, int d_model) {
    __shared__ f32x4 sums[32][8];
    const int c = threadIdx.x % 8, g = threadIdx.x / 8;
    const int col = blockIdx.x * 32 + c * 4;                        // of dw and dbias side by side
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (col < 2 * d_model) {
#pragma unroll 8
        for (int i = g; i < parts; i += 32) v += *reinterpret_cast<const f32x4*>(part + (size_t)i * 2 * d_model + col);
    }
    sums[g][c] = v;
    __syncthreads();
    if (g == 0 && col < 2 * d_model) {
#pragma unroll
        for (int i = 1; i < 32; ++i) v += sums[i][c];
        uint16_t* to = col < d_model ? dw + col : db ? db + (col - d_model) : nullptr;
        if (to) st_global_8(to, u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])});
    }
}

// ------------------------------------------------------------------------------------------
namespace {
template <class F>
void with_shape(int d_model, F go) {
    using row_ops::Shape;
    if (d_model <= 64) go(Shape<8, 1, 1>{});
    else if (d_model <= 128) go(Shape<16, 1, 1>{});
    else if (d_model <= 256) go(Shape<32, 1, 1>{});
    else if (d_model <= 512) go(Shape<64, 1, 1>{});
    else if (d_model <= 1024) go(Shape<64, 1, 2>{});
    else if (d_model <= 2048) go(Shape<64, 2, 2>{});
    else if (d_model <= 4096) go(Shape<64, 4, 2>{});
    else go(Shape<64, 8, 2>{});
}
// Of the backward: one piece a lane; five and ten waves to a row where eight and sixteen would leave many without work, as the RMS norm's.
template <class F>
void with_bwd_shape(int d_model, F go) {
    using row_ops::Shape;
    if (d_model <= 64) go(Shape<8, 1, 1>{});
    else if (d_model <= 128) go(Shape<16, 1, 1>{});
    else if (d_model <= 256) go(Shape<32, 1, 1>{});
    else if (d_model <= 512) go(Shape<64, 1, 1>{});
    else if (d_model <= 1024) go(Shape<64, 2, 1>{});
    else if (d_model <= 2048) go(Shape<64, 4, 1>{});
    else if (d_model <= 2560) go(Shape<64, 5, 1>{});
    else if (d_model <= 4096) go(Shape<64, 8, 1>{});
    else if (d_model <= 5120) go(Shape<64, 10, 1>{});
    else go(Shape<64, 16, 1>{});
}
constexpr size_t ALONE = 2;                                          // so many groups of rows at most are one workgroup's, which then has dw
template <class S>
size_t bwd_parts(size_t rows) {
    constexpr int ROWS = 1024 / (S::LPR * S::WPR);
    const size_t groups = (rows + ROWS - 1) / ROWS, most = groups <= ALONE ? 1 : 256;
    return groups < most ? groups : most;
}
}  // namespace

bool layernorm_residual_fits(size_t rows, int d_model) {
    bool fits = false;
    with_shape(d_model, [&](auto shape) {
        using S = decltype(shape);
        fits = (rows + S::ROWS - 1) / S::ROWS * S::THREADS < ((size_t)1 << 32);
    });
    return fits;
}

int launch_layernorm_residual(const void* x, const void* residual, const void* weight, const void* bias, void* out,
                              void* out_resid, size_t rows, int d_model, float eps, hipStream_t stream) {
    const bool cached = rows * d_model * (residual ? 8 : 4) <= kStreamCached;
    with_shape(d_model, [&](auto shape) {
        using S = decltype(shape);
        auto go = [&](auto in_cache, auto with_res, auto with_bias) {
            launch_kernel((layernorm_residual_kernel<S, in_cache(), with_res(), with_bias()>), dim3((unsigned)((rows + S::ROWS - 1) / S::ROWS)),
                          dim3(S::THREADS), 0, stream, static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(residual),
                          static_cast<const uint16_t*>(weight), static_cast<const uint16_t*>(bias), static_cast<uint16_t*>(out),
                          static_cast<uint16_t*>(out_resid), rows, d_model, eps, out == x);
        };
        auto pick = [&](auto in_cache) {
            if (residual) { if (bias) go(in_cache, std::true_type{}, std::true_type{}); else go(in_cache, std::true_type{}, std::false_type{}); }
            else { if (bias) go(in_cache, std::false_type{}, std::true_type{}); else go(in_cache, std::false_type{}, std::false_type{}); }
        };
        if (cached) pick(std::true_type{}); else pick(std::false_type{});
    });
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

size_t layernorm_residual_bwd_workspace_bytes(size_t rows, int d_model) {
    size_t parts = 0;
    with_bwd_shape(d_model, [&](auto shape) { parts = bwd_parts<decltype(shape)>(rows); });
    return parts * 2 * d_model * sizeof(float);
}

int launch_layernorm_residual_bwd(const void* d_out, const void* d_resid, const void* resid, const void* weight, void* dx, void* dweight,
                                  void* dbias, size_t rows, int d_model, float eps, void* workspace, hipStream_t stream) {
    const bool cached = rows * d_model * (d_resid ? 8 : 6) <= kStreamCached;
    size_t parts = 0;
    with_bwd_shape(d_model, [&](auto shape) {
        using S = decltype(shape);
        parts = bwd_parts<S>(rows);
        constexpr int ROWS = 1024 / (S::LPR * S::WPR);
        const size_t lds = (size_t)(ROWS / 2) * 2 * d_model * sizeof(float);    // at most 32 KB
        auto go = [&](auto in_cache, auto with_resid) {
            launch_kernel((layernorm_residual_bwd_kernel<S, in_cache(), with_resid()>), dim3((unsigned)parts), dim3(S::LPR * S::WPR * ROWS), lds, stream,
                          static_cast<const uint16_t*>(d_out), static_cast<const uint16_t*>(d_resid), static_cast<const uint16_t*>(resid),
                          static_cast<const uint16_t*>(weight), static_cast<uint16_t*>(dx), static_cast<float*>(workspace),
                          parts == 1 ? static_cast<uint16_t*>(dweight) : nullptr, parts == 1 ? static_cast<uint16_t*>(dbias) : nullptr, rows, d_model, eps);
        };
        if (d_resid) { if (cached) go(std::true_type{}, std::true_type{}); else go(std::false_type{}, std::true_type{}); }
        else { if (cached) go(std::true_type{}, std::false_type{}); else go(std::false_type{}, std::false_type{}); }
    });
    if (hipGetLastError() != hipSuccess) return -1;
    if (parts == 1) return 0;
    launch_kernel(layernorm_dweight_kernel, dim3((unsigned)((2 * d_model + 31) / 32)), dim3(256), 0, stream, static_cast<const float*>(workspace),
                  static_cast<uint16_t*>(dweight), static_cast<uint16_t*>(dbias), (int)parts, d_model);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tyr
