// A key-value cache in pages (gfx950): writing new tokens into it, and attention of one new token over it.
//
// The pools k_pages and v_pages are [num_pages][Hkv][page_size][D], bf16 or e4m3 (then K = k_scale[kv head] * the stored value, V
// alike).  Row j of sequence b is row j % page_size of page page_table[b][j / page_size].  A page size is a multiple of 16, so the
// 16 rows of an MFMA tile lie in one page; an entry outside [0, num_pages) is a page that is not there.
//
// Attention.  Row j of a sequence of n rows is visible iff j < n and (no window, or j >= n - window, or j < sinks).  The visible
// rows are walked as a list of 16-row tiles, the sinks' first; pages without a visible row are never looked at.
//   grid: one workgroup per (piece of a sequence, kv head, block of 16 of its query heads).  How a batch is cut into pieces is
//   decided on the device from the lengths that are there, by every workgroup for itself: pieces of `chunk` tiles, so that there are
//   about `target` workgroups however the lengths are spread and however wide the table is, and a captured launch follows lengths
//   that change between replays.  The host only bounds the grid, (B + target / heads) pieces a head.
//   Partial results (O, m, l) of sequences of several pieces are joined by a second launch, as
//     m = max m_s ; l = sum l_s 2^(m_s-m) ; O = sum O_s 2^(m_s-m) / l ; LSE = ln l + m ln 2.
// HBM-bound: each visible row of K and V is read once a block of query heads, straight into MFMA operand registers (16x16x32 bf16):
//   S^T (16 rows x 16 q) = K x Q^T and O^T_j (16 d x 16 q) += V^T x P^T, j = 0..7, the layouts of the contiguous decode:
//   lane l = (x = l % 16, g = l / 16) holds row x of K and, of V, the columns 8x..8x+7 of the rows 4g..4g+3 whose probabilities the
//   accumulator of S^T leaves in it, so P^T needs no movement; V is transposed 8x8 in registers.
//   P is given as bf16 twice, its rounding and what that left: products with the second cost matrix time that is idle here, and
//   the result is as exact as with f32 probabilities.
#include "common.hpp"
#include "launch.hpp"

namespace tyr {

namespace paged {
constexpr int TILE = 16, WAVES = 4, THREADS = 64 * WAVES, QPAD = 16;
constexpr int MIN_CHUNK = 8;                // tiles of a piece at least
constexpr int TARGET = 512;                 // pieces times heads that a launch aims at
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
};
__device__ __forceinline__ int rows_of(const int* kv_lens, int b, int cap) { return max(0, min(kv_lens[b], cap)); }

struct Piece { int b, split, splits, first; };   // sequence; which of its pieces; pieces of sequences before it; b < 0: none

// Piece j of the batch.  Every wave works it out for itself, 64 sequences at a time.
__device__ __forceinline__ Piece find_piece(const int* kv_lens, int B, int cap, int window, int sinks, int heads, int target, int j, int lane) {
    uint64_t tiles = 0;
    for (int b = lane; b < B; b += 64) tiles += Rows(rows_of(kv_lens, b, cap), window, sinks).count;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) tiles += __shfl_xor(tiles, o, 64);
    const uint64_t even = (tiles * heads + target - 1) / target;
    const int chunk = (int)max((uint64_t)MIN_CHUNK, min(even, (uint64_t)1 << 28));       // a sequence has less than 2^27 tiles
    int before = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int b = b0 + lane;
        const int mine = b < B ? max(1, (Rows(rows_of(kv_lens, b, cap), window, sinks).count + chunk - 1) / chunk) : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int left = __shfl_up(upto, o, 64);
            if (lane >= o) upto += left;
        }
        const int first = before + upto - mine;
        const uint64_t here = __builtin_amdgcn_ballot_w64(j >= first && j < first + mine);
        if (here) {
            const int at = __builtin_ctzll(here);
            const int start = __builtin_amdgcn_readlane(first, at);
            return {b0 + at, j - start, __builtin_amdgcn_readlane(mine, at), start};
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return {-1, 0, 0, 0};
}

struct Args {
    const uint16_t* q;
    const void *k, *v;
    const int *table, *kv_lens;
    const float *k_scale, *v_scale;
    uint16_t* o;
    float *lse, *part_o, *part_m, *part_l;
    int2* plan;                             // [B] first piece and pieces of each sequence
    int B, Hq, Hkv, G, blocks;              // G = query heads of a kv head; blocks of 16 of them
    int width, page_tiles, pages;           // pages of a table row; tiles of a page; pages of the pool
    int cap, window, sinks, target;
    float scale_log2;
};

// What a lane holds of 32 rows.
template <int D, bool FP8> struct Buf {
    u32x4 k[2][D / 32];                     // [T][i]: row x of tile T, d = 32i + 8g + [0,8)
    u32x4 v[8];                             // [p]: row 4g + p%4 of tile p/4, d = 8 (x mod D/8) + [0,8)
};
template <int D> struct Buf<D, true> {
    u32x4 k[2][D / 64];                     // [T][c]: row x of tile T, d = 16 (4c + g) + [0,16)
    u32x2 v[8];
};

__device__ __forceinline__ uint32_t bf16_of_e4m3(uint32_t four, bool upper) {
    const bf16x2 r = upper ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, 1.0f, false);
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ u32x4 bf16_of_e4m3(uint32_t lo, uint32_t hi) {
    return u32x4{bf16_of_e4m3(lo, false), bf16_of_e4m3(lo, true), bf16_of_e4m3(hi, false), bf16_of_e4m3(hi, true)};
}
}  // namespace paged

template <int D, bool FP8>
__global__ __launch_bounds__(paged::THREADS) void paged_decode_kernel(const paged::Args a) {
    using namespace paged;
    extern __shared__ __attribute__((aligned(16))) float smem[];   // [WAVES][heads][D] O, then [WAVES][QPAD] m, l
    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), x = lane & 15, g = lane >> 4;
    const int heads = a.Hkv * a.blocks;
    const int hb = (int)(blockIdx.x % (unsigned)heads), j = (int)(blockIdx.x / (unsigned)heads);
    const int kvh = hb / a.blocks, q0 = (hb % a.blocks) * 16, nq = min(16, a.G - q0);     // query heads q0 .. q0 + nq of kv head kvh
    Piece piece{j, 0, 1, j};
    if (a.target) {
        piece = find_piece(a.kv_lens, a.B, a.cap, a.window, a.sinks, heads, a.target, j, lane);
        if (piece.b < 0) return;
        if (hb == 0 && piece.split == 0 && t == 0) a.plan[piece.b] = int2{piece.first, piece.splits};
    }
    const int b = piece.b;
    const Rows rows(rows_of(a.kv_lens, b, a.cap), a.window, a.sinks);
    const int c0 = (int)((int64_t)rows.count * piece.split / piece.splits), c1 = (int)((int64_t)rows.count * (piece.split + 1) / piece.splits);

    // Q^T operand: column x = query head q0 + x (zero beyond the block's heads)
    constexpr int KI = D / 32, ES = FP8 ? 1 : 2;
    const size_t head0 = (size_t)b * a.Hq + (size_t)kvh * a.G + q0;
    bf16x8 qf[KI];
    {
        const uint16_t* qp = a.q + (head0 + min(x, nq - 1)) * D;
#pragma unroll
        for (int i = 0; i < KI; ++i) {
            const int d = FP8 ? 16 * (4 * (i >> 1) + g) + 8 * (i & 1) : 32 * i + 8 * g;
            u32x4 v = ld_global_16(qp + d);
            if (x >= nq) v = u32x4{0, 0, 0, 0};
            qf[i] = __builtin_bit_cast(bf16x8, v);
        }
    }
    const float scale_log2 = a.scale_log2 * (a.k_scale ? a.k_scale[kvh] : 1.0f);

    f32x4 oacc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) oacc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m2 = -INFINITY, lsum = 0.0f;

    // The waves take the piece's 32-row steps in turn.  Where a step's two tiles are and which of their rows count is worked out by
    // the lanes for 32 steps at once (lane 2s + T: tile T of step s), and read from them as scalars.
    const int nsteps = max(0, ((c1 - c0 + 1) / 2 - w + WAVES - 1) / WAVES);
    const int* entries = a.table + (size_t)b * a.width;
    struct Where { int tile; uint32_t mask; };
    auto locate = [&](int step0) {
        const int i = c0 + 2 * (w + WAVES * (step0 + (lane >> 1))) + (lane & 1);
        Where r{0, 0};
        if (i < c1) {
            const int tile = rows.tile(i), page = tile / a.page_tiles, id = entries[page];
            if (id >= 0 && id < a.pages) r = {(id * a.Hkv + kvh) * a.page_tiles + tile - page * a.page_tiles, rows.mask(tile)};
        }
        return r;
    };
    Where at[2] = {locate(0), Where{0, 0}};
    if (nsteps > 32) at[1] = locate(32);

    auto load = [&](Buf<D, FP8>& bf, int st) {
        const int from = st & 32 ? at[1].tile : at[0].tile;
#pragma unroll
        for (int T = 0; T < 2; ++T) {
            const size_t base = (size_t)(uint32_t)__builtin_amdgcn_readlane(from, 2 * (st & 31) + T) * (TILE * D * ES);
            const unsigned char *kb = static_cast<const unsigned char*>(a.k) + base, *vb = static_cast<const unsigned char*>(a.v) + base;
            if constexpr (FP8) {
#pragma unroll
                for (int c = 0; c < D / 64; ++c) bf.k[T][c] = ld_global_16_nt(kb + x * D + 16 * (4 * c + g));
#pragma unroll
                for (int p = 0; p < 4; ++p)
                    bf.v[4 * T + p] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(vb + (4 * g + p) * D + (x & (D / 8 - 1)) * 8));
            } else {
#pragma unroll
                for (int i = 0; i < KI; ++i) bf.k[T][i] = ld_global_16_nt(kb + (x * D + 32 * i + 8 * g) * 2);
#pragma unroll
                for (int p = 0; p < 4; ++p) bf.v[4 * T + p] = ld_global_16_nt(vb + ((4 * g + p) * D + (x & (D / 8 - 1)) * 8) * 2);
            }
        }
    };

    auto compute = [&](const Buf<D, FP8>& bf, int st) {
        const uint32_t masks = st & 32 ? at[1].mask : at[0].mask;
        uint32_t seen[2];
        f32x4 sacc[2];
        u32x4 v[8];
#pragma unroll
        for (int T = 0; T < 2; ++T) {
            seen[T] = (uint32_t)__builtin_amdgcn_readlane((int)masks, 2 * (st & 31) + T);
            sacc[T] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < KI; ++i) {
                u32x4 k;
                if constexpr (FP8) k = i & 1 ? bf16_of_e4m3(bf.k[T][i / 2][2], bf.k[T][i / 2][3]) : bf16_of_e4m3(bf.k[T][i / 2][0], bf.k[T][i / 2][1]);
                else k = bf.k[T][i];
                sacc[T] = mfma_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), qf[i], sacc[T]);
            }
        }
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            if constexpr (FP8) v[p] = bf16_of_e4m3(bf.v[p][0], bf.v[p][1]);
            else v[p] = bf.v[p];
        }
        // register r of tile T is its row 4g + r.  What is hidden may hold anything: its score goes, and its V, which 0 * NaN would keep.
        if ((seen[0] & seen[1]) != 0xffffu) {
#pragma unroll
            for (int T = 0; T < 2; ++T)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!(seen[T] >> (4 * g + r) & 1)) {
                        sacc[T][r] = -INFINITY;
                        v[4 * T + r] = u32x4{0, 0, 0, 0};
                    }
        }
        float mx = fmaxf(fmaxf(fmaxf(sacc[0][0], sacc[0][1]), fmaxf(sacc[0][2], sacc[0][3])),
                         fmaxf(fmaxf(sacc[1][0], sacc[1][1]), fmaxf(sacc[1][2], sacc[1][3])));
        mx = max_xor32(max_xor16(mx));
        const float m2new = fmaxf(m2, mx * scale_log2);
        const float ref = m2new == -INFINITY ? 0.0f : m2new;       // nothing seen yet: every power below is of -inf
        const float alpha = fast_exp2(m2 - ref);
        if (__builtin_amdgcn_ballot_w64(m2new > m2) != 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) oacc[i] *= alpha;
        }
        m2 = m2new;
        float pv[8], psum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            pv[i] = fast_exp2(fmaf(sacc[i >> 2][i & 3], scale_log2, -ref));
            psum += pv[i];
        }
        lsum = lsum * alpha + psum;
        u32x4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            hi[i] = pack_bf16(pv[2 * i], pv[2 * i + 1]);
            lo[i] = pack_bf16(pv[2 * i] - bf16_lo(hi[i]), pv[2 * i + 1] - bf16_hi(hi[i]));
        }
        u32x4 vt[8];
        transpose8x8_b16(v, vt);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            oacc[i] = mfma_16x16x32_bf16(__builtin_bit_cast(bf16x8, vt[i]), __builtin_bit_cast(bf16x8, hi), oacc[i]);
            oacc[i] = mfma_16x16x32_bf16(__builtin_bit_cast(bf16x8, vt[i]), __builtin_bit_cast(bf16x8, lo), oacc[i]);
        }
    };

    Buf<D, FP8> b0, b1;
    if (nsteps > 0) load(b0, 0);
#pragma unroll
    for (int i = 0; i < KI; ++i) pin_registers(qf[i]);
    for (int st = 0; st < nsteps; st += 2) {
        if (st + 1 < nsteps) load(b1, st + 1);
        compute(b0, st);
        if (st + 1 < nsteps) {
            if (st + 2 < nsteps) load(b0, st + 2);
            compute(b1, st + 1);
        }
        // the half that steps st+2 on do not need takes the places of 32 steps further on
        if (((st + 2) & 31) == 0 && st + 2 + 32 < nsteps) at[(st >> 5) & 1] = locate(st + 2 + 32);
    }

    // ---- merge the waves through LDS.  oacc[i][r] is O^T[d = 32g + 8r + i][q = x].
    float* so = smem;                                // [WAVES][nq][D]
    float* sm = smem + WAVES * nq * D;               // [WAVES][QPAD]
    float* sl = sm + WAVES * QPAD;
    const float ltot = sum_xor32(sum_xor16(lsum));
    if (x < nq && 32 * g < D) {
        float* dst = so + ((size_t)w * nq + x) * D + 32 * g;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            *reinterpret_cast<f32x4*>(dst + 8 * r) = f32x4{oacc[0][r], oacc[1][r], oacc[2][r], oacc[3][r]};
            *reinterpret_cast<f32x4*>(dst + 8 * r + 4) = f32x4{oacc[4][r], oacc[5][r], oacc[6][r], oacc[7][r]};
        }
    }
    if (x < nq && g == 0) { sm[w * QPAD + x] = m2; sl[w * QPAD + x] = ltot; }
    __syncthreads();
    const float v_scale = a.v_scale ? a.v_scale[kvh] : 1.0f;
    const int per = min(16, a.G);                    // partial slots are laid out for this many heads
    for (int idx = t; idx < nq * D; idx += THREADS) {
        const int qh = idx / D, d = idx % D;
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) m = fmaxf(m, sm[i * QPAD + qh]);
        const float ref = m == -INFINITY ? 0.0f : m;
        float o = 0.0f, l = 0.0f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            const float wgt = fast_exp2(sm[i * QPAD + qh] - ref);       // of a wave that saw no row: 0, and so are its sums
            o += so[((size_t)i * nq + qh) * D + d] * wgt;
            l += sl[i * QPAD + qh] * wgt;
        }
        o *= v_scale;
        if (piece.splits == 1) {
            a.o[(head0 + qh) * D + d] = (uint16_t)(pack_bf16(l == 0.0f ? 0.0f : o / l, 0.0f) & 0xffffu);
            if (d == 0 && a.lse) a.lse[head0 + qh] = l == 0.0f ? -INFINITY : logf(l) + m * LN2;
        } else {
            const size_t at_part = (size_t)blockIdx.x * per + qh;
            a.part_o[at_part * D + d] = o;
            if (d == 0) { a.part_m[at_part] = m; a.part_l[at_part] = l; }
        }
    }
}

// Joins the pieces of a sequence: one workgroup per (sequence, query head), D/4 threads of 4 elements a piece, several side by side.
template <int D>
__global__ __launch_bounds__(256) void paged_join_kernel(const paged::Args a) {
    using namespace paged;
    constexpr int TPS = D / 4, CG = 256 / TPS;
    __shared__ f32x4 so[CG][TPS];
    __shared__ float sm[CG], sl[CG];
    const int b = blockIdx.x / (unsigned)a.Hq, qh = blockIdx.x % (unsigned)a.Hq;
    const int2 plan = a.plan[b];
    const int S = plan.y;
    if (S < 2) return;
    const int t = threadIdx.x, c = t % TPS, sg = t / TPS;
    const int kvh = qh / a.G, inner = qh % a.G, hb = kvh * a.blocks + inner / 16, per = min(16, a.G), heads = a.Hkv * a.blocks;
    const size_t slot0 = ((size_t)plan.x * heads + hb) * per + inner % 16, pitch = (size_t)heads * per;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;
    for (int s0 = sg; s0 < S; s0 += 4 * CG) {
        f32x4 os[4];
        float ms[4], ls[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const size_t slot = slot0 + min(s0 + i * CG, S - 1) * pitch;
            ms[i] = s0 + i * CG < S ? a.part_m[slot] : -INFINITY;
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
            if (s0 + i * CG < S) {
                const float wgt = fast_exp2(ms[i] - ref);
                o += os[i] * wgt;
                l += ls[i] * wgt;
            }
    }
    so[sg][c] = o;
    if (c == 0) { sm[sg] = m; sl[sg] = l; }
    __syncthreads();
    if (t >= TPS) return;
    const int n = min(CG, S);
    for (int i = 1; i < n; ++i) {
        const float mn = fmaxf(m, sm[i]), ref = mn == -INFINITY ? 0.0f : mn, f = fast_exp2(m - ref), wgt = fast_exp2(sm[i] - ref);
        o = o * f + so[i][c] * wgt;
        l = l * f + sl[i] * wgt;
        m = mn;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const size_t head = (size_t)b * a.Hq + qh;
    reinterpret_cast<u32x2*>(a.o + head * D)[c] = u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
    if (a.lse && c == 0) a.lse[head] = l == 0.0f ? -INFINITY : logf(l) + m * LN2;
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

// One thread takes 8 elements of each half of one head of one token; heads of a token: Hq of q, Hkv of k, Hkv of v.
template <bool FP8>
__global__ __launch_bounds__(256) void paged_rope_append_kernel(const paged::AppendArgs a) {
    using namespace paged;
    const uint32_t id = blockIdx.x * 256u + threadIdx.x;
    if (id >= a.threads) return;
    const unsigned per_head = a.D / 16, per_token = (a.Hq + 2 * a.Hkv) * per_head;
    const unsigned token = id / per_token, rest = id - token * per_token, head = rest / per_head;
    const int e0 = (int)(rest - head * per_head) * 8, half = a.D / 2;
    const int b = (int)(token / (unsigned)a.T), step = (int)(token - (unsigned)b * a.T);
    const int first = a.positions[b];
    const int64_t pos = (int64_t)first + step;
    const bool rotated = first >= 0 && pos < a.rope_rows;
    const int hk = (int)head - a.Hq;                       // < 0: a query head; < Hkv: of k; else of v
    const uint16_t* src = hk < 0 ? a.q + ((size_t)token * a.Hq + head) * a.D
                          : hk < a.Hkv ? a.k_new + ((size_t)token * a.Hkv + hk) * a.D : a.v_new + ((size_t)token * a.Hkv + hk - a.Hkv) * a.D;
    const u32x4 lo = ld_global_16(src + e0), hi = ld_global_16(src + half + e0);
    float x1[8], x2[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x1[2 * i] = bf16_lo(lo[i]), x1[2 * i + 1] = bf16_hi(lo[i]);
        x2[2 * i] = bf16_lo(hi[i]), x2[2 * i + 1] = bf16_hi(hi[i]);
    }
    if (rotated && hk < a.Hkv) rotate8(x1, x2, a.cos + (size_t)pos * half + e0, a.sin + (size_t)pos * half + e0);
    auto pack = [](const float (&f)[8]) { return u32x4{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])}; };
    if (hk < 0) {
        uint16_t* to = a.q_out + ((size_t)token * a.Hq + head) * a.D + e0;
        st_global_16(to, rotated ? pack(x1) : u32x4{0, 0, 0, 0});
        st_global_16(to + half, rotated ? pack(x2) : u32x4{0, 0, 0, 0});
        return;
    }
    if (!rotated || (a.new_lens && step >= a.new_lens[b])) return;
    const int64_t page = pos / a.page_size;
    if (page >= a.width) return;
    const int entry = a.table[(size_t)b * a.width + page];
    if (entry < 0 || entry >= a.pages) return;
    const bool is_v = hk >= a.Hkv;
    const int kvh = is_v ? hk - a.Hkv : hk;
    const size_t at = (((size_t)entry * a.Hkv + kvh) * a.page_size + (size_t)(pos - page * a.page_size)) * a.D + e0;
    void* pool = is_v ? a.v_pages : a.k_pages;
    if constexpr (FP8) {
        const float* scales = is_v ? a.v_scale : a.k_scale;
        const float s = scales ? scales[kvh] : 1.0f;
        auto pack8 = [s](const float (&f)[8]) {
            return u32x2{pack_e4m3(f32x4{f[0] / s, f[1] / s, f[2] / s, f[3] / s}), pack_e4m3(f32x4{f[4] / s, f[5] / s, f[6] / s, f[7] / s})};
        };
        st_global_8(static_cast<uint8_t*>(pool) + at, pack8(x1));
        st_global_8(static_cast<uint8_t*>(pool) + at + half, pack8(x2));
    } else {
        st_global_16(static_cast<uint16_t*>(pool) + at, pack(x1));
        st_global_16(static_cast<uint16_t*>(pool) + at + half, pack(x2));
    }
}

// ------------------------------------------------------------------------------------------
namespace {
struct Grid { int heads, per, target; uint64_t pieces; };      // blocks of heads; heads of a slot; 0 = a piece a sequence; workgroups
Grid paged_grid(int64_t B, int Hq, int Hkv, int64_t cap) {
    const int G = Hq / Hkv, heads = Hkv * ((G + 15) / 16);
    // sequences that cannot be longer than one piece are not cut (and not joined)
    const int target = cap <= paged::MIN_CHUNK * paged::TILE ? 0 : paged::TARGET;
    return {heads, G < 16 ? G : 16, target, (uint64_t)B * heads + target};
}
}  // namespace

uint64_t paged_decode_workgroups(int B, int Hq, int Hkv, int64_t cap) { return paged_grid(B, Hq, Hkv, cap).pieces; }

size_t paged_decode_workspace_bytes(int B, int Hq, int Hkv, int D, int64_t cap) {
    const Grid g = paged_grid(B, Hq, Hkv, cap);
    if (!g.target) return 0;
    return (size_t)g.pieces * g.per * (D + 2) * sizeof(float) + ((size_t)B * sizeof(int2) + 15) / 16 * 16;
}

int launch_paged_decode(const void* q, const void* k_pages, const void* v_pages, const int* page_table, const int* kv_lens,
                        const float* k_scale, const float* v_scale, void* o, float* lse, int B, int Hq, int Hkv, int D, int pages,
                        int page_size, int width, int window, int sinks, int e4m3, float scale, void* workspace, hipStream_t stream) {
    using namespace paged;
    const Grid g = paged_grid(B, Hq, Hkv, (int64_t)width * page_size);
    Args a{};
    a.q = static_cast<const uint16_t*>(q);
    a.k = k_pages, a.v = v_pages;
    a.table = page_table, a.kv_lens = kv_lens;
    a.k_scale = k_scale, a.v_scale = v_scale;
    a.o = static_cast<uint16_t*>(o), a.lse = lse;
    if (g.target) {
        a.plan = static_cast<int2*>(workspace);
        a.part_o = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + ((size_t)B * sizeof(int2) + 15) / 16 * 16);
        a.part_m = a.part_o + (size_t)g.pieces * g.per * D;
        a.part_l = a.part_m + (size_t)g.pieces * g.per;
    }
    a.B = B, a.Hq = Hq, a.Hkv = Hkv, a.G = Hq / Hkv, a.blocks = (a.G + 15) / 16;
    a.width = width, a.page_tiles = page_size / TILE, a.pages = pages;
    a.cap = width * page_size, a.window = window, a.sinks = sinks, a.target = g.target;
    a.scale_log2 = scale * LOG2E;
    const size_t lds = (size_t)(WAVES * g.per * D + 2 * WAVES * QPAD) * sizeof(float);       // at most 33 KB
    const dim3 grid((unsigned)g.pieces);
    auto kernel = D == 128 ? (e4m3 ? &paged_decode_kernel<128, true> : &paged_decode_kernel<128, false>)
                           : (e4m3 ? &paged_decode_kernel<64, true> : &paged_decode_kernel<64, false>);
    launch_kernel(kernel, grid, dim3(THREADS), lds, stream, a);
    if (hipGetLastError() != hipSuccess) return -1;
    if (!g.target) return 0;
    launch_kernel(D == 128 ? &paged_join_kernel<128> : &paged_join_kernel<64>, dim3((unsigned)((size_t)B * Hq)), dim3(256), 0, stream, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

int launch_paged_rope_append(const void* q, const void* k_new, const void* v_new, const float* cosp, const float* sinp, void* q_out,
                             void* k_pages, void* v_pages, const int* page_table, const int* positions, const int* new_lens,
                             const float* k_scale, const float* v_scale, int B, int T, int Hq, int Hkv, int D, int pages, int page_size,
                             int width, int rope_rows, int e4m3, hipStream_t stream) {
    paged::AppendArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k_new), static_cast<const uint16_t*>(v_new), cosp, sinp,
                        static_cast<uint16_t*>(q_out), k_pages, v_pages, page_table, positions, new_lens, k_scale, v_scale,
                        T, Hq, Hkv, D, pages, page_size, width, rope_rows, (uint32_t)((uint64_t)B * T * (Hq + 2 * Hkv) * (D / 16))};
    launch_kernel(e4m3 ? &paged_rope_append_kernel<true> : &paged_rope_append_kernel<false>, dim3((a.threads + 255u) / 256u), dim3(256), 0, stream, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tyr
