// A key-value cache in pages (gfx950): writing new tokens into it, and attention of one new token over it.
//
// The pools k_pages and v_pages are [num_pages][Hkv][page_size][D], bf16 or e4m3 (then K = k_scale[kv head] * the stored value, V
// alike).  Row j of sequence b is row j % page_size of page page_table[b][j / page_size].  A page size is a multiple of 16, so the
// 16 rows of an MFMA tile lie in one page; an entry outside [0, num_pages) is a page that is not there.
//
// Attention.  Row j of a sequence of n rows is visible iff j < n and (no window, or j >= n - window, or j < sinks).  The visible
// rows are walked as a list of 16-row tiles, the sinks' first, two tiles a step; pages without a visible row are never looked at.
//   All steps of all heads (a head: one kv head of one sequence, and a block of its query heads) stand in one row, sequence by
//   sequence, and are dealt out evenly to as many waves as the device holds, one a SIMD: each works out its share from the lengths
//   that are there, so neither unequal lengths nor a table much wider than they are leave CUs idle, and a captured launch follows
//   lengths that change between replays.  A wave goes through its share without a pause between heads.  (Workgroups of four waves on
//   one piece of a sequence, joined through LDS, 512 and more of them: 64 sequences of 37 to 32768 e4m3 rows took 160-190 us, 116 so;
//   32 sequences of 8192 bf16 rows 182, 172 so.)
//   Heads that several waves have a part of are joined by a second launch from partial results (O, m, l), as
//     m = max m_s ; l = sum l_s 2^(m_s-m) ; O = sum O_s 2^(m_s-m) / l ; LSE = ln l + m ln 2.
// HBM-bound: each visible row of K and V is read once a block of 16 query heads, or two, straight into MFMA operand registers (16x16x32 bf16):
//   S^T (16 rows x 16 q) = K x Q^T and O^T_j (16 d x 16 q) += V^T x P^T, j = 0..7, the layouts of the contiguous decode:
//   lane l = (x = l % 16, g = l / 16) holds row x of K and, of V, the columns 8x..8x+7 of the rows 4g..4g+3 whose probabilities the
//   accumulator of S^T leaves in it, so P^T needs no movement; V is transposed 8x8 in registers.
//   P is given as bf16 twice, its rounding and what that left (below 2^-16 of it is lost): products with the second cost matrix time that
//   is idle here, and the result is as exact as with f32 probabilities.
#include "common.hpp"
#include "launch.hpp"

#include <algorithm>
#include <type_traits>

namespace tyr {

namespace paged {
constexpr int TILE = 16, STEP = 2 * TILE;
constexpr int SHARES = 1024;                // waves that share a launch's steps: one on every SIMD of 256 CUs
constexpr int MIN_SHARE = 2;                // steps of a wave at least
constexpr int WHOLE = 8;                    // sequences of so many steps at most are not cut, and so need no join: 88 heads of 6 steps 7.5 us whole, 8.8
                                            // cut; of 8 8.7, 9.0; 1024 heads of 8 23.2, 25.4; 32 heads of 10 9.6, 8.0
// More than 16 query heads of a kv head are several blocks.  Where each block is a head of its own, its rows come from memory once a block.
// Two other ways have them come once for two blocks, or for all:
//   - a wave takes two blocks (bf16 rows of 128 leave no registers for that).  Its steps take longer, so only launches that have many of
//     them, by their tables' width: 128 sequences of 8192 e4m3 rows, 32 query heads of one kv head 98.7 us, 63 so; 64 of 4000 29.1, 30.4.
constexpr int WIDE = 32768;                 // steps of all blocks from which
//   - waves side by side in a workgroup take a block each of the same steps and keep together by a barrier, so that all but the first find
//     the rows in the caches: bf16 rows of 128 where sequences are cut.  128 sequences of 8192 rows, 32 heads 182 us, 118 so (1024 shares
//     124, and without the barrier 162); 28 of 2517 24.6, 19.0; 96 of 5 steps, not cut, 6.7, 7.4; 128 of 8192 e4m3 rows 98.7, 94.2.
constexpr int SIDE_BY_SIDE = 8;             // of them at most: as many as have their registers on a CU at once
constexpr int TURN = 3;                     // steps that going from one head to the next is counted as
constexpr int MANY_HEADS = 64;              // heads of a launch from which one wave joins each, not four (1024 heads of 3-22 steps 40.7 us, 37.4 so;
                                            // with 8 heads of 128 parts four waves have more of them under way)
constexpr int LONG = 32;                    // parts of a head up to which that is so
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// The visible rows of a sequence as a list of tiles.
struct Rows {
    int n, lo, sinks;                       // rows; first row of the window; rows before it that stay visible
    int sink_tiles, first;                  // tiles before the window's; the window's first tile
    int count;                              // tiles in all
    __device__ __forceinline__ Rows(int n_, int window, int sinks_) {
        n = n_;
        lo = window > 0 ? max(0, n - window) : 0;
        sinks = min(sinks_, lo);
        first = lo / TILE;
        sink_tiles = min((sinks + TILE - 1) / TILE, first);
        count = sink_tiles + (n + TILE - 1) / TILE - first;
    }
    __device__ __forceinline__ int tile(int i) const { return i < sink_tiles ? i : i - sink_tiles + first; }
    // bit r: row r of tile t is visible
    __device__ __forceinline__ uint32_t mask(int t) const {
        auto below = [t](int row) { return (1u << max(0, min(TILE, row - t * TILE))) - 1u; };
        return below(n) & (~below(lo) | below(sinks));
    }
    // of 32 rows; a sequence without rows has one, in which nothing is visible, and so gets its zeros written
    __device__ __forceinline__ int steps() const { return max(1, (count + 1) / 2); }
};

// Sum of x over this lane and those before it, by moves of the vector unit.
__device__ __forceinline__ int sum_upto(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);      // 1, 2, 4, 8 lanes to the left in rows of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);      // lane 15 of a row to rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);      // lane 31 to rows 2 and 3
    return x;
}

struct Args {
    const uint16_t* q;
    const void *k, *v;
    const int *table, *kv_lens;
    const float *k_scale, *v_scale;
    uint16_t* o;
    float *lse, *part_o, *part_m, *part_l;
    int2* plan;                             // [B] first step of each sequence's first head, steps of a head; [B]: steps of a wave, of the longest head
    int B, Hq, Hkv, G;                      // G = query heads of a kv head
    int per, apart, beside;                 // query heads of a block; blocks that are heads of their own; blocks of waves side by side
    int width, page_tiles, pages;           // pages of a table row; tiles of a page; pages of the pool
    int cap, window, sinks, shares;         // shares = 0: every wave takes one head of one sequence, nothing is cut
    float scale_log2;
};

// The sequences in rounds of 64, one a lane.
struct Round {
    int b0, n, steps, upto;                 // its first sequence; this lane's rows, steps of a head, and those (and turns) up to it in the round
    __device__ __forceinline__ void read(const Args& a, int b0_, int lane) {
        b0 = b0_;
        const int b = b0 + lane;
        n = b < a.B ? max(0, min(a.kv_lens[b], a.cap)) : 0;
        steps = b < a.B ? Rows(n, a.window, a.sinks).steps() : 0;
        upto = sum_upto(b < a.B ? steps + TURN : 0);
    }
    __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(upto, 63); }
};

// A factor that is the same for all lanes, by a scalar load: one more vector load that may be under way at the end of a branch would have the
// compiler wait there, in every step, for all the rows asked for since.
__device__ __forceinline__ float factor(const float* scales, int i) {
    return scales ? *reinterpret_cast<const __attribute__((address_space(4))) float*>(reinterpret_cast<uintptr_t>(scales + i)) : 1.0f;
}

// What a lane holds of 32 rows.
template <int D, bool FP8> struct Buf {
    u32x4 k[2][D / 32];                     // [T][i]: row x of tile T, d = 32i + 8g + [0,8)
    u32x4 v[8];                             // [p]: row 4g + p%4 of tile p/4, d = 8 (x mod D/8) + [0,8)
};
template <int D> struct Buf<D, true> {
    u32x4 k[2][D / 64];                     // [T][c]: row x of tile T, d = 16 (4c + g) + [0,16)
    u32x2 v[8];
};

// A tile of a pool as a buffer of `bytes` bytes.  Of one of no bytes loads give 0 and read nothing, so every step loads alike,
// also behind the last one: a load that may or may not have been made is one that the compiler waits for together with all later ones.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* pool, size_t at, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(pool) + at), 0, bytes, 0x00020000);
}
// AGAIN: waves beside this one read the same.  Else the caches are not to keep it (32 sequences of 8192 rows 172 us, 195 if they do).
template <bool AGAIN> __device__ __forceinline__ u32x4 load_tile_16(__amdgpu_buffer_rsrc_t t, int at) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(t, at, 0, AGAIN ? 0 : 2));
}
template <bool AGAIN> __device__ __forceinline__ u32x2 load_tile_8(__amdgpu_buffer_rsrc_t t, int at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(t, at, 0, AGAIN ? 0 : 2));
}

__device__ __forceinline__ float last_bit_set(float x) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) | 1u); }

__device__ __forceinline__ uint32_t bf16_of_e4m3(uint32_t four, bool upper) {
    const bf16x2 r = upper ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, 1.0f, false);
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ u32x4 bf16_of_e4m3(uint32_t lo, uint32_t hi) {
    return u32x4{bf16_of_e4m3(lo, false), bf16_of_e4m3(lo, true), bf16_of_e4m3(hi, false), bf16_of_e4m3(hi, true)};
}
}  // namespace paged

// QB: 16 query heads or 32 of a wave.  AGAIN: a workgroup is a.beside waves side by side, else one (of four, a launch with few waves would
// have them on fewer CUs: one sequence of 1500 rows 8.8 us, 10.2 so).
template <int D, bool FP8, int QB, bool AGAIN>
__global__ __launch_bounds__(64 * (AGAIN ? paged::SIDE_BY_SIDE : 1), 2) void paged_decode_kernel(const paged::Args a) {
    using namespace paged;
    const int lane = threadIdx.x & 63, x = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(AGAIN ? blockIdx.x * a.beside + threadIdx.x / 64 : blockIdx.x));
    const int place = AGAIN ? blockIdx.x : wave;     // which share of the steps
    const int side = AGAIN ? __builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64)) : 0;
    const int heads = a.Hkv * a.apart;
    constexpr int KI = D / 32, TILE_BYTES = TILE * D * (FP8 ? 1 : 2);

    // ---- this wave's steps [at, end) of all, and the head of the sequence in which they begin
    Round round;
    int at, end, b, hb, first;                       // first = the sequence's (head's) first step
    if (a.shares == 0) {
        b = place / heads;
        hb = place - b * heads;
        round.read(a, b & ~63, lane);
        at = first = 0;
        end = __builtin_amdgcn_readlane(round.steps, b & 63);
    } else {
        round.read(a, 0, lane);
        int all = round.total();
        if (a.B > 64) {
            int more = 0;
#pragma unroll 4
            for (int i = 64 + lane; i < a.B; i += 64) more += Rows(max(0, min(a.kv_lens[i], a.cap)), a.window, a.sinks).steps() + TURN;
            all += __builtin_amdgcn_readlane(sum_upto(more), 63);
        }
        all *= heads;
        const int share = max(MIN_SHARE, (all + a.shares - 1) / a.shares);
        // one wave more than there are shares writes down the plan, for the launch that joins
        const bool scribe = place == a.shares;
        if (scribe && side > 0) return;
        int longest = 0;                                 // steps of a head
        at = min((int64_t)place * share, (int64_t)all);
        end = min(at + share, all);
        if (!scribe && at >= end) return;
        // the round in which step `at` lies
        int base = 0;
        for (;;) {
            const int upto = base + round.total() * heads, b0 = round.b0 + lane;
            if (scribe) {
                if (b0 < a.B) a.plan[b0] = int2{base + (round.upto - round.steps - TURN) * heads, round.steps};
                longest = max(longest, round.steps);
            } else if (at < upto) break;
            base = upto;
            if (round.b0 + 64 >= a.B) break;
            round.read(a, round.b0 + 64, lane);
        }
        if (scribe) {
            for (int d = 32; d > 0; d /= 2) longest = max(longest, __shfl_xor(longest, d));
            if (lane == 0) a.plan[a.B] = int2{share, longest};
            return;
        }
        // the first lane whose sequence ends behind `at`; none if the lengths changed under the two readings of them
        const uint64_t behind = __builtin_amdgcn_ballot_w64(at < base + round.upto * heads);
        if (behind == 0 || at < base) return;
        const int i = __builtin_ctzll(behind);
        const int each = __builtin_amdgcn_readlane(round.steps, i) + TURN;
        const int start = base + (__builtin_amdgcn_readlane(round.upto, i) - each) * heads;
        b = round.b0 + i;
        hb = (at - start) / each;
        first = start + hb * each;
    }

    // ---- where the rows of a step are.  The lanes work it out for up to 32 steps of one head at once (lane 2s + T: tile T of step s).
    struct Run { int tile; uint32_t mask; int steps, b, hb, first, last; };       // steps of the run; the head's first step and its end
    int next_at = at, next_b = b, next_hb = hb, next_first = first;
    auto turn = [&]() {                              // to the next head
        next_first += __builtin_amdgcn_readlane(round.steps, next_b - round.b0) + TURN;
        next_at = next_first;
        if (++next_hb == heads) {
            next_hb = 0;
            if (++next_b - round.b0 == 64) round.read(a, next_b, lane);
            if (next_b >= a.B) next_at = end;        // the lengths changed: no sequence is left
        }
    };
    auto locate = [&]() {
        Run r;
        const Rows rows(__builtin_amdgcn_readlane(round.n, next_b - round.b0), a.window, a.sinks);
        r.b = next_b, r.hb = next_hb, r.first = next_first;
        r.last = next_first + rows.steps();
        r.steps = min(32, min(r.last, end) - next_at);
        r.tile = 0, r.mask = 0;
        const int t = 2 * (next_at - next_first) + lane;
        if (t < rows.count && lane < 2 * r.steps) {
            const int tile = rows.tile(t), page = tile / a.page_tiles, id = a.table[(size_t)next_b * a.width + page];
            if (id >= 0 && id < a.pages) {
                r.tile = (id * a.Hkv + next_hb / a.apart) * a.page_tiles + tile - page * a.page_tiles;
                r.mask = rows.mask(tile);
            }
        }
        next_at += r.steps;
        if (next_at == r.last && next_at < end) turn();
        return r;
    };
    if (at - first >= __builtin_amdgcn_readlane(round.steps, b - round.b0)) {       // the wave's share begins in a turn
        turn();
        if (next_at >= end) return;
        b = next_b, hb = next_hb, first = next_first;
    }

    struct Slot { Buf<D, FP8> buf; uint32_t seen[2]; int b, hb, first, last, live; };
    Run run = locate(), then = run;
    then.steps = 0;
    int s = 0;                                       // step of the run to load next
    auto load = [&](Slot& o) {
        if (s >= run.steps) {
            run = then;
            s = 0;
            then.steps = 0;
            if (next_at < end) then = locate();
        }
        o.live = __builtin_amdgcn_readfirstlane(run.steps);      // 0: there was no step left
        o.b = run.b, o.hb = run.hb, o.first = run.first, o.last = run.last;
#pragma unroll
        for (int T = 0; T < 2; ++T) {
            o.seen[T] = (uint32_t)__builtin_amdgcn_readlane((int)run.mask, 2 * s + T);
            const size_t base = (size_t)(uint32_t)__builtin_amdgcn_readlane(run.tile, 2 * s + T) * TILE_BYTES;
            const int there = o.live > 0 && o.seen[T] ? TILE_BYTES : 0;
            const auto k = tile_rsrc(a.k, base, there), v = tile_rsrc(a.v, base, there);
            if constexpr (FP8) {
#pragma unroll
                for (int c = 0; c < D / 64; ++c) o.buf.k[T][c] = load_tile_16<AGAIN>(k, x * D + 16 * (4 * c + g));
#pragma unroll
                for (int p = 0; p < 4; ++p) o.buf.v[4 * T + p] = load_tile_8<AGAIN>(v, (4 * g + p) * D + (x & (D / 8 - 1)) * 8);
            } else {
#pragma unroll
                for (int i = 0; i < KI; ++i) o.buf.k[T][i] = load_tile_16<AGAIN>(k, (x * D + 32 * i + 8 * g) * 2);
#pragma unroll
                for (int p = 0; p < 4; ++p) o.buf.v[4 * T + p] = load_tile_16<AGAIN>(v, ((4 * g + p) * D + (x & (D / 8 - 1)) * 8) * 2);
            }
        }
        ++s;
    };

    // ---- one head: Q^T operand (column x = query head q0 + x, zero beyond the block's heads) and running sums
    __shared__ u32x4 qs[AGAIN ? SIDE_BY_SIDE : 1][QB * KI][64];
    u32x4 (&qf)[QB * KI][64] = qs[side];      // a lane reads what it wrote: registers are short, LDS is idle
    f32x4 oacc[QB][8];
    float m2[QB], lsum[QB], scale_log2;
    int nq, kvh;
    size_t head0;
    auto begin = [&](int b_, int hb_) {
        kvh = hb_ / a.apart;
        const int q0 = (AGAIN ? side : hb_ - kvh * a.apart) * (16 * QB);
        nq = min(16 * QB, a.G - q0);
        head0 = (size_t)b_ * a.Hq + (size_t)kvh * a.G + q0;
#pragma unroll
        for (int c = 0; c < QB; ++c) {
            const uint16_t* qp = a.q + (head0 + min(16 * c + x, nq - 1)) * D;
#pragma unroll
            for (int i = 0; i < KI; ++i) {
                u32x4 v = ld_global_16(qp + (FP8 ? 16 * (4 * (i >> 1) + g) + 8 * (i & 1) : 32 * i + 8 * g));
                if (16 * c + x >= nq) v = u32x4{0, 0, 0, 0};
                qf[c * KI + i][lane] = v;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) oacc[c][i] = f32x4{0.f, 0.f, 0.f, 0.f};
            m2[c] = -INFINITY;
            lsum[c] = 0.0f;
        }
        scale_log2 = a.scale_log2 * factor(a.k_scale, kvh);
    };
    // The head's steps are done, or this wave's: its result where the wave had all of them, else a partial one.  A wave has at most two
    // heads that it shares with others: one that began before it, and one that goes on behind it.  oacc[i][r] is O^T[d = 32g + 8r + i][x].
    auto finish = [&](int first_, int last_) {
        const float v_scale = factor(a.v_scale, kvh);
#pragma unroll
        for (int c = 0; c < QB; ++c) {
            const float l = sum_xor32(sum_xor16(lsum[c]));
            const int h = 16 * c + x;
            if (h >= nq || 32 * g >= D) continue;
            const f32x4 (&o)[8] = oacc[c];
            if (first_ >= at && last_ <= end) {
                const float f = l == 0.0f ? 0.0f : v_scale / l;
                uint16_t* to = a.o + (head0 + h) * D + 32 * g;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    st_global_16(to + 8 * r, u32x4{pack_bf16(o[0][r] * f, o[1][r] * f), pack_bf16(o[2][r] * f, o[3][r] * f),
                                                   pack_bf16(o[4][r] * f, o[5][r] * f), pack_bf16(o[6][r] * f, o[7][r] * f)});
                if (g == 0 && a.lse) a.lse[head0 + h] = l == 0.0f ? -INFINITY : logf(l) + m2[c] * LN2;
            } else {
                const size_t slot = (size_t)(2 * wave + (first_ < at ? 0 : 1)) * min(16 * QB, a.G) + h;
                float* to = a.part_o + slot * D + 32 * g;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    *reinterpret_cast<f32x4*>(to + 8 * r) = f32x4{o[0][r], o[1][r], o[2][r], o[3][r]} * v_scale;
                    *reinterpret_cast<f32x4*>(to + 8 * r + 4) = f32x4{o[4][r], o[5][r], o[6][r], o[7][r]} * v_scale;
                }
                if (g == 0) { a.part_m[slot] = m2[c]; a.part_l[slot] = l; }
            }
        }
    };

    int now = first, now_last = 0;                   // the head whose sums are in the registers
    auto compute = [&](const Slot& o) {
        if (o.first != now) {
            finish(now, now_last);
            begin(o.b, o.hb);
            now = o.first;
        }
        now_last = o.last;
        f32x4 sacc[QB][2];
        u32x4 v[8];
#pragma unroll
        for (int T = 0; T < 2; ++T) {
#pragma unroll
            for (int c = 0; c < QB; ++c) sacc[c][T] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < KI; ++i) {
                u32x4 k;
                if constexpr (FP8) k = i & 1 ? bf16_of_e4m3(o.buf.k[T][i / 2][2], o.buf.k[T][i / 2][3]) : bf16_of_e4m3(o.buf.k[T][i / 2][0], o.buf.k[T][i / 2][1]);
                else k = o.buf.k[T][i];
#pragma unroll
                for (int c = 0; c < QB; ++c)
                    sacc[c][T] = mfma_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), __builtin_bit_cast(bf16x8, qf[c * KI + i][lane]), sacc[c][T]);
            }
        }
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            if constexpr (FP8) v[p] = bf16_of_e4m3(o.buf.v[p][0], o.buf.v[p][1]);
            else v[p] = o.buf.v[p];
        }
#pragma unroll
        for (int c = 0; c < QB; ++c)                 // before anything is hidden: the pages' factor may be 0 or negative
#pragma unroll
            for (int T = 0; T < 2; ++T) sacc[c][T] *= scale_log2;
        // register r of tile T is its row 4g + r.  What is hidden may hold anything: its score goes, and its V, which 0 * NaN would keep.
        if ((o.seen[0] & o.seen[1]) != 0xffffu) {
#pragma unroll
            for (int T = 0; T < 2; ++T)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!(o.seen[T] >> (4 * g + r) & 1)) {
#pragma unroll
                        for (int c = 0; c < QB; ++c) sacc[c][T][r] = -INFINITY;
                        v[4 * T + r] = u32x4{0, 0, 0, 0};
                    }
        }
        u32x4 hi[QB], lo[QB];
#pragma unroll
        for (int c = 0; c < QB; ++c) {
            const f32x4 (&sc)[2] = sacc[c];
            float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])), fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
            mx = max_xor32(max_xor16(mx));
            const float m2new = fmaxf(m2[c], mx);
            const float ref = m2new == -INFINITY ? 0.0f : m2new;       // nothing seen yet: every power below is of -inf
            const float alpha = fast_exp2(m2[c] - ref);
            if (__builtin_amdgcn_ballot_w64(m2new > m2[c]) != 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) oacc[c][i] *= alpha;
            }
            m2[c] = m2new;
            float pv[8], psum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                pv[i] = fast_exp2(sc[i >> 2][i & 3] - ref);
                psum += pv[i];
            }
            lsum[c] = lsum[c] * alpha + psum;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (FP8) {
                    hi[c][i] = pack_bf16(pv[2 * i], pv[2 * i + 1]);
                } else {
                    // bf16 V may be infinite, so both parts of a probability are positive: the first rounded down, the other not 0 (the
                    // least bit of the 24 is set).  Rounded to nearest, the other is 0 or negative half of the time, and inf + 0 inf is NaN.
                    pv[2 * i] = last_bit_set(pv[2 * i]);
                    pv[2 * i + 1] = last_bit_set(pv[2 * i + 1]);
                    hi[c][i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, pv[2 * i + 1]), __builtin_bit_cast(uint32_t, pv[2 * i]), 0x07060302u);
                }
                lo[c][i] = pack_bf16(pv[2 * i] - bf16_lo(hi[c][i]), pv[2 * i + 1] - bf16_hi(hi[c][i]));
            }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {                // columns 2n and 2n + 1 of V's 8x8 piece, transposed
            u32x4 even, odd;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                even[i] = __builtin_amdgcn_perm(v[2 * i + 1][n], v[2 * i][n], 0x05040100u);
                odd[i] = __builtin_amdgcn_perm(v[2 * i + 1][n], v[2 * i][n], 0x07060302u);
            }
#pragma unroll
            for (int c = 0; c < QB; ++c) {
                oacc[c][2 * n] = mfma_16x16x32_bf16(__builtin_bit_cast(bf16x8, even), __builtin_bit_cast(bf16x8, hi[c]), oacc[c][2 * n]);
                oacc[c][2 * n] = mfma_16x16x32_bf16(__builtin_bit_cast(bf16x8, even), __builtin_bit_cast(bf16x8, lo[c]), oacc[c][2 * n]);
                oacc[c][2 * n + 1] = mfma_16x16x32_bf16(__builtin_bit_cast(bf16x8, odd), __builtin_bit_cast(bf16x8, hi[c]), oacc[c][2 * n + 1]);
                oacc[c][2 * n + 1] = mfma_16x16x32_bf16(__builtin_bit_cast(bf16x8, odd), __builtin_bit_cast(bf16x8, lo[c]), oacc[c][2 * n + 1]);
            }
        }
    };

    Slot s0, s1;                                     // the rows of one step are under way while those of the other are in use
    load(s0);
    begin(b, hb);
    if (next_at < end) then = locate();
    // One way out, behind both halves' loads: with one between them the compiler would take s1's for the last ones made, and wait for
    // s0's with them.
    do {
        if constexpr (AGAIN) __builtin_amdgcn_s_barrier();       // the waves side by side ask for the same rows together
        load(s1);
        compute(s0);
        if constexpr (AGAIN) __builtin_amdgcn_s_barrier();
        load(s0);
        if (s1.live) compute(s1);
    } while (s0.live);
    finish(now, now_last);
}

namespace paged {
// The parts of a query head: the partial results of the waves that had some of its steps.
struct Parts {
    int w0, S, beside, inner;               // the first of the waves, their number; which of the waves side by side; the head's place in its block
    size_t head;
    __device__ __forceinline__ Parts(const Args& a, int b, int qh) {
        const int2 plan = a.plan[b];
        const int share = a.plan[a.B].x;
        const int kvh = qh / a.G, block = a.per < a.G ? (qh - kvh * a.G) / a.per : 0;
        inner = qh - kvh * a.G - block * a.per;
        const int hb = a.apart > 1 ? kvh * a.apart + block : kvh;
        beside = a.beside > 1 ? block : 0;
        const int first = plan.x + hb * (plan.y + TURN);
        w0 = first / share;
        S = min((first + plan.y - 1) / share, a.shares - 1) - w0 + 1;
        head = (size_t)b * a.Hq + qh;
    }
    // of the first wave: the head that goes on behind it; of the others the one that began before them
    __device__ __forceinline__ size_t slot(const Args& a, int i) const { return (size_t)(2 * ((w0 + i) * a.beside + beside) + (i == 0 ? 1 : 0)) * a.per + inner; }
};
// Four elements of O, and m and l, of parts g, g + groups, ...: four under way at a time.
struct Sum { f32x4 o; float m, l; };
template <int D>
__device__ __forceinline__ Sum join_every(const Args& a, const Parts& p, int c, int g, int groups) {
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;
    for (int s0 = g; s0 < p.S; s0 += 4 * groups) {
        f32x4 os[4];
        float ms[4], ls[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const size_t slot = p.slot(a, min(s0 + i * groups, p.S - 1));
            ms[i] = s0 + i * groups < p.S ? a.part_m[slot] : -INFINITY;
            ls[i] = a.part_l[slot];
            os[i] = *reinterpret_cast<const f32x4*>(a.part_o + slot * D + 4 * c);
        }
        const float mn = fmaxf(fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3])), m), ref = mn == -INFINITY ? 0.0f : mn;
        const float alpha = fast_exp2(m - ref);
        o *= alpha;
        l *= alpha;
        m = mn;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s0 + i * groups < p.S) {
                const float wgt = fast_exp2(ms[i] - ref);
                o += os[i] * wgt;
                l += ls[i] * wgt;
            }
    }
    return Sum{o, m, l};
}
template <int D>
__device__ __forceinline__ void store_head(const Args& a, const Parts& p, int c, const Sum& t) {
    const float inv = t.l == 0.0f ? 0.0f : 1.0f / t.l;
    reinterpret_cast<u32x2*>(a.o + p.head * D)[c] = u32x2{pack_bf16(t.o[0] * inv, t.o[1] * inv), pack_bf16(t.o[2] * inv, t.o[3] * inv)};
    if (a.lse && c == 0) a.lse[p.head] = t.l == 0.0f ? -INFINITY : logf(t.l) + t.m * LN2;
}
// A head by a workgroup of 256 threads: D/4 threads of 4 elements a part, several parts side by side.
template <int D> struct Side { f32x4 o[1024 / D][D / 4]; float m[1024 / D], l[1024 / D]; };
template <int D>
__device__ __forceinline__ void join_by_all(const Args& a, const Parts& p, Side<D>& side) {
    constexpr int TPS = D / 4, CG = 256 / TPS;
    const int t = threadIdx.x, c = t % TPS, g = t / TPS;
    Sum x = join_every<D>(a, p, c, g, CG);
    side.o[g][c] = x.o;
    if (c == 0) { side.m[g] = x.m; side.l[g] = x.l; }
    __syncthreads();
    if (t >= TPS) return;
    const int n = min(CG, p.S);
    for (int i = 1; i < n; ++i) {
        const float mn = fmaxf(x.m, side.m[i]), ref = mn == -INFINITY ? 0.0f : mn, f = fast_exp2(x.m - ref), wgt = fast_exp2(side.m[i] - ref);
        x.o = x.o * f + side.o[i][c] * wgt;
        x.l = x.l * f + side.l[i] * wgt;
        x.m = mn;
    }
    store_head<D>(a, p, c, x);
}
}  // namespace paged

// Joins the parts of a head: one workgroup per (sequence, query head).  It is all latency, 3-4 us (m, l and the weights of 64 parts by the
// lanes of a wave instead, no serial step: as long).
template <int D>
__global__ __launch_bounds__(256) void paged_join_kernel(const paged::Args a) {
    using namespace paged;
    __shared__ Side<D> side;
    const Parts p(a, blockIdx.x / (unsigned)a.Hq, blockIdx.x % (unsigned)a.Hq);
    if (p.S >= 2) join_by_all<D>(a, p, side);
}

// The same with a wave a head, for launches of many heads, most of which have few parts.  Where the longest head has more than LONG, what has
// more is one for all waves of a workgroup after all, in workgroups far apart, so that the heads of a sequence do not wait for each other.  64
// heads of 8 query heads each, one of 100000 rows and 63 of 20: 35.8 us, 84.8 with a wave for each; 64 of 1 to 32768 rows 33.0, 39.2.  It
// costs 0.9 of 73 us where 2048 short sequences are joined.
template <int D>
__global__ __launch_bounds__(256) void paged_join_few_kernel(const paged::Args a) {
    using namespace paged;
    constexpr int TPS = D / 4, CG = 64 / TPS;
    __shared__ Side<D> side;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64)), id = blockIdx.x * 4 + wave;
    const int b = id / a.Hq, lane = threadIdx.x & 63;
    const Parts p(a, min(b, a.B - 1), id - b * a.Hq);
    const int S = b < a.B ? p.S : 0;
    const int2 all = a.plan[a.B];
    const bool far = all.y > all.x * (LONG - 2);                  // the same for the whole launch
    if (S >= 2 && !(far && S > LONG)) {
        const int c = lane % TPS, g = lane / TPS;
        Sum x = join_every<D>(a, p, c, g, CG);
        // the groups of lanes together
        float m = max_xor32(x.m);
        if constexpr (CG == 4) m = max_xor16(m);
        const float f = fast_exp2(x.m - (m == -INFINITY ? 0.0f : m));
        auto sum = [&](float y) {
            y = sum_xor32(y * f);
            if constexpr (CG == 4) y = sum_xor16(y);
            return y;
        };
        x.m = m;
        x.l = sum(x.l);
#pragma unroll
        for (int i = 0; i < 4; ++i) x.o[i] = sum(x.o[i]);
        if (g == 0) store_head<D>(a, p, c, x);
    }
    if (!far) return;
    for (int i = blockIdx.x; i < a.B * a.Hq; i += gridDim.x) {    // at most four
        const Parts of(a, i / a.Hq, i % a.Hq);
        if (of.S <= LONG) continue;
        join_by_all<D>(a, of, side);
        __syncthreads();                                          // the next one writes what this one reads
    }
}

// ---- new tokens into the pages ---------------------------------------------------------------
namespace paged {
struct AppendArgs {
    const uint16_t *q, *k_new, *v_new;
    const float *cos, *sin;
    uint16_t* q_out;
    void *k_pages, *v_pages;
    const int *table, *positions, *new_lens;
    const float *k_scale, *v_scale;
    int T, Hq, Hkv, D, pages, page_size, width, rope_rows;
    uint32_t threads;
};
// y1 = x1 cos - x2 sin, y2 = x1 sin + x2 cos of 8 elements of each half, as the rotary kernels of this library: separate products and sum
__device__ __forceinline__ void rotate8(float (&x1)[8], float (&x2)[8], const float* c, const float* s) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma clang fp contract(off)
        const float y1 = x1[i] * c[i] - x2[i] * s[i], y2 = x1[i] * s[i] + x2[i] * c[i];
        x1[i] = y1;
        x2[i] = y2;
    }
}
}  // namespace paged

// One thread takes 8 elements of each half of one head of one token; heads of a token: Hq of q, Hkv of k, Hkv of v.  What bounds it is
// memory, and where little is moved the chain position -> page -> store; the elements are asked for before it begins.  (Several heads a
// thread, so that the rotary table's 64 bytes and the page are looked up once for all: 2222 tokens of 48 heads 12.3 us, 13.1 with
// two heads, 16.5 with four.)
template <bool FP8>
__global__ __launch_bounds__(256) void paged_rope_append_kernel(const paged::AppendArgs a) {
    using namespace paged;
    const uint32_t id = blockIdx.x * 256u + threadIdx.x;
    if (id >= a.threads) return;
    const unsigned per_head = a.D / 16, per_token = (a.Hq + 2 * a.Hkv) * per_head;
    const unsigned token = id / per_token, rest = id - token * per_token;
    unsigned head = rest / per_head;
    const int e0 = (int)(rest - head * per_head) * 8, half = a.D / 2;
    const int b = (int)(token / (unsigned)a.T), step = (int)(token - (unsigned)b * a.T);
    const int kind = head < (unsigned)a.Hq ? 0 : head < (unsigned)(a.Hq + a.Hkv) ? 1 : 2;     // q, k, v
    const unsigned heads = kind ? a.Hkv : a.Hq;
    head -= kind ? a.Hq + (kind - 1) * a.Hkv : 0;
    const uint16_t* src = (kind == 0 ? a.q : kind == 1 ? a.k_new : a.v_new) + ((size_t)token * heads + head) * a.D + e0;
    const u32x4 lo = ld_global_16(src), hi = ld_global_16(src + half);
    const int first = a.positions[b], lens = a.new_lens ? a.new_lens[b] : a.T;
    const bool placed = first >= 0 && (int64_t)first + step < a.rope_rows;
    const unsigned pos = (unsigned)first + step;
    float x1[8], x2[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x1[2 * i] = bf16_lo(lo[i]), x1[2 * i + 1] = bf16_hi(lo[i]);
        x2[2 * i] = bf16_lo(hi[i]), x2[2 * i + 1] = bf16_hi(hi[i]);
    }
    if (kind < 2 && placed) rotate8(x1, x2, a.cos + (size_t)pos * half + e0, a.sin + (size_t)pos * half + e0);
    auto pack = [](const float (&f)[8]) { return u32x4{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])}; };
    if (kind == 0) {
        uint16_t* to = a.q_out + ((size_t)token * heads + head) * a.D + e0;
        st_global_16_nt(to, placed ? pack(x1) : u32x4{0, 0, 0, 0});
        st_global_16_nt(to + half, placed ? pack(x2) : u32x4{0, 0, 0, 0});
        return;
    }
    if (!placed || step >= lens) return;
    const unsigned page = pos / (unsigned)a.page_size;
    if (page >= (unsigned)a.width) return;
    const int entry = a.table[(size_t)b * a.width + page];
    if (entry < 0 || entry >= a.pages) return;
    const size_t at = (((size_t)entry * a.Hkv + head) * a.page_size + (pos - page * a.page_size)) * a.D + e0;
    void* pool = kind == 2 ? a.v_pages : a.k_pages;
    if constexpr (FP8) {
        const float* scales = kind == 2 ? a.v_scale : a.k_scale;
        const float f = scales ? scales[head] : 1.0f;
        // x / f, rounded as a division is: the product with the rounded reciprocal, and what it left, once more (infinite ones stay);
        // 16 divisions took 1 us of 11
        const float rf = 1.0f / f;
        auto over = [f, rf](float x) {
            const float y = x * rf;
            return fabsf(y) < INFINITY ? fmaf(fmaf(-y, f, x), rf, y) : y;
        };
        auto pack8 = [over](const float (&x)[8]) {
            return u32x2{pack_e4m3(f32x4{over(x[0]), over(x[1]), over(x[2]), over(x[3])}), pack_e4m3(f32x4{over(x[4]), over(x[5]), over(x[6]), over(x[7])})};
        };
        st_global_8(static_cast<uint8_t*>(pool) + at, pack8(x1));
        st_global_8(static_cast<uint8_t*>(pool) + at + half, pack8(x2));
    } else {
        st_global_16_nt(static_cast<uint16_t*>(pool) + at, pack(x1));
        st_global_16_nt(static_cast<uint16_t*>(pool) + at + half, pack(x2));
    }
}

// ------------------------------------------------------------------------------------------
namespace {
struct Grid { int per, apart, beside, shares; uint64_t groups; };         // as in Args; workgroups of the launch
Grid paged_grid(int64_t B, int Hq, int Hkv, int D, int e4m3, int64_t cap, int64_t window, int64_t sinks) {
    using namespace paged;
    // a window and the sinks may each begin and end inside a tile
    const int64_t rows = window > 0 ? std::min(cap, window + 2 * TILE + sinks + 2 * TILE) : cap;
    const int64_t steps = std::max<int64_t>(1, (rows + STEP - 1) / STEP);
    const int G = Hq / Hkv;
    Grid g{std::min(G, 16), (G + 15) / 16, 1, 0, 0};
    if (G > 16) {
        if (D == 128 && !e4m3) {
            if (steps > WHOLE && g.apart <= SIDE_BY_SIDE) g.beside = g.apart, g.apart = 1;
        } else if (B * Hkv * g.apart * steps >= WIDE) {
            g.per = std::min(G, 32), g.apart = (G + 31) / 32;
        }
    }
    g.groups = (uint64_t)B * Hkv * g.apart;
    if (steps > WHOLE) {
        const int64_t most = g.beside == 1 ? SHARES : std::min(SHARES / 2, 256 * (8 / g.beside));
        g.shares = (int)std::min<int64_t>(most, ((int64_t)g.groups * (steps + TURN) + MIN_SHARE - 1) / MIN_SHARE);
        g.groups = g.shares + 1;
    }
    return g;
}
size_t plan_bytes(int B) { return ((size_t)(B + 1) * sizeof(int2) + 15) / 16 * 16; }
}  // namespace

size_t paged_decode_workspace_bytes(int B, int Hq, int Hkv, int D, int64_t cap) {
    size_t most = 0;                                        // of both formats; a window makes it no more
    for (int e4m3 = 0; e4m3 < 2; ++e4m3) {
        const Grid g = paged_grid(B, Hq, Hkv, D, e4m3, cap, 0, 0);
        if (g.shares) most = std::max(most, plan_bytes(B) + (size_t)g.shares * g.beside * 2 * g.per * (D + 2) * sizeof(float));
    }
    return most;
}

int launch_paged_decode(const void* q, const void* k_pages, const void* v_pages, const int* page_table, const int* kv_lens,
                        const float* k_scale, const float* v_scale, void* o, float* lse, int B, int Hq, int Hkv, int D, int pages,
                        int page_size, int width, int window, int sinks, int e4m3, float scale, void* workspace, hipStream_t stream) {
    using namespace paged;
    const Grid g = paged_grid(B, Hq, Hkv, D, e4m3, (int64_t)width * page_size, window, sinks);
    Args a{};
    a.q = static_cast<const uint16_t*>(q);
    a.k = k_pages, a.v = v_pages;
    a.table = page_table, a.kv_lens = kv_lens;
    a.k_scale = k_scale, a.v_scale = v_scale;
    a.o = static_cast<uint16_t*>(o), a.lse = lse;
    if (g.shares) {
        a.plan = static_cast<int2*>(workspace);
        const size_t slots = (size_t)g.shares * g.beside * 2 * g.per;
        a.part_o = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + plan_bytes(B));
        a.part_m = a.part_o + slots * D;
        a.part_l = a.part_m + slots;
    }
    a.B = B, a.Hq = Hq, a.Hkv = Hkv, a.G = Hq / Hkv;
    a.per = g.per, a.apart = g.apart, a.beside = g.beside;
    a.width = width, a.page_tiles = page_size / TILE, a.pages = pages;
    a.cap = width * page_size, a.window = window, a.sinks = sinks, a.shares = g.shares;
    a.scale_log2 = scale * LOG2E;
    auto pick = [&](auto qb) {
        return D == 128 ? &paged_decode_kernel<128, true, qb(), false> : e4m3 ? &paged_decode_kernel<64, true, qb(), false> : &paged_decode_kernel<64, false, qb(), false>;
    };
    auto kernel = D == 128 && !e4m3 ? (g.beside > 1 ? &paged_decode_kernel<128, false, 1, true> : &paged_decode_kernel<128, false, 1, false>)
                                    : g.per > 16 ? pick(std::integral_constant<int, 2>{}) : pick(std::integral_constant<int, 1>{});
    launch_kernel(kernel, dim3((unsigned)g.groups), dim3(64 * g.beside), 0, stream, a);
    if (hipGetLastError() != hipSuccess) return -1;
    if (!g.shares) return 0;
    const size_t heads = (size_t)B * Hq;
    if ((int64_t)B * Hkv * g.apart * g.beside < MANY_HEADS)
        launch_kernel(D == 128 ? &paged_join_kernel<128> : &paged_join_kernel<64>, dim3((unsigned)heads), dim3(256), 0, stream, a);
    else
        launch_kernel(D == 128 ? &paged_join_few_kernel<128> : &paged_join_few_kernel<64>, dim3((unsigned)((heads + 3) / 4)), dim3(256), 0, stream, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

int launch_paged_rope_append(const void* q, const void* k_new, const void* v_new, const float* cosp, const float* sinp, void* q_out,
                             void* k_pages, void* v_pages, const int* page_table, const int* positions, const int* new_lens,
                             const float* k_scale, const float* v_scale, int B, int T, int Hq, int Hkv, int D, int pages, int page_size,
                             int width, int rope_rows, int e4m3, hipStream_t stream) {
    paged::AppendArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k_new), static_cast<const uint16_t*>(v_new), cosp, sinp,
                        static_cast<uint16_t*>(q_out), k_pages, v_pages, page_table, positions, new_lens, k_scale, v_scale,
                        T, Hq, Hkv, D, pages, page_size, width, rope_rows, (uint32_t)((uint64_t)B * T * (Hq + 2 * Hkv) * (D / 16))};
    auto kernel = e4m3 ? &paged_rope_append_kernel<true> : &paged_rope_append_kernel<false>;
    launch_kernel(kernel, dim3((a.threads + 255u) / 256u), dim3(256), 0, stream, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tyr
