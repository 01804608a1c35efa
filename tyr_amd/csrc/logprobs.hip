// Log probabilities of given tokens, with entropy and the largest alternatives, and their gradient (gfx950).
//
// Of a row x of `vocab` logits, m its largest, s = sum e^(x - m), t = sum (x - m) e^(x - m):
//   lse = m + ln s,   logp = x[target] - m - ln s,   entropy = ln s - t / s,   alternatives: the `top` largest x, equal ones by place.
// Gradient, with p = e^(x - lse) and the gradients of logp, entropy and lse that arrive:
//   dx = p (d_lse - d_logp - d_entropy (ln p + entropy)) + d_logp [at the target]
//
// One pass over the row: every lane keeps m, s and t of its own elements and scales them when its m grows; they are joined at the end, in f32.
// The alternatives need no second pass: the `top`-th largest of the lanes' m is no larger than the `top`-th largest element.  Every lane keeps
// the maxima of its blocks of 64 bytes, too, and only the blocks that reach that limit are read once more (all of such a lane's elements:
// each 16 bytes of them another cache line, with 20 alternatives nearly the whole row again, 4096 x 50001 108 us, 80 so).
//
// Bound by HBM (bf16: and nearly by the vector units, 7 to 9 instructions an element, of which the exponential counts as four).
//
// A row begins at any element: up to 16 bytes' worth at its two ends are taken one by one, what lies between in pieces of 16 bytes.
#include <algorithm>
#include <type_traits>

#include "launch.hpp"
#include "rows.hpp"

namespace tyr {

namespace lp {
constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int AT_ONCE = 4;                        // pieces a lane asks for together
constexpr int BWD_THREADS = 256, BWD_AT_ONCE = 2; // of the gradient
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;
constexpr float LEAST = -3.402823466e38f;         // m of no element: the smallest finite number
constexpr float TAME = 1024.0f;                   // size of m up to which an element's exponent is one multiplication and addition
constexpr int MAX_TOP = 64;
constexpr int KEPT = 512;                         // candidates that stay when the list is cut
constexpr int TURN = 128;                         // threads that add to it in a turn
constexpr int LIST = KEPT + TURN * 8;
constexpr int SLOTS = 16;                         // maxima of blocks a thread; block b is in slot b % SLOTS
constexpr int MOST_BLOCKS = 1024;
constexpr int JOINED = 256;                       // alternatives of all parts together that the join looks for its limit among

template <class T> struct Elem;
template <> struct Elem<uint16_t> {
    static constexpr int E = 8;
    static __device__ __forceinline__ float one(uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = bf16_lo(v[i]); f[2 * i + 1] = bf16_hi(v[i]); }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
        return u32x4{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])};
    }
    static __device__ __forceinline__ void put(uint16_t* p, float v) { *p = (uint16_t)pack_bf16(v, 0.0f); }
};
template <> struct Elem<float> {
    static constexpr int E = 4;
    static __device__ __forceinline__ float one(float v) { return v; }
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[4]) {
        const f32x4 x = __builtin_bit_cast(f32x4, v);              // (a bit cast of one element of a vector reads the first)
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = x[i];
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[4]) {
        return __builtin_bit_cast(u32x4, f32x4{f[0], f[1], f[2], f[3]});
    }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};

// A stretch of a row, [begin, end) in elements of the row: `head` single elements, `pieces` of E, `tail` single ones.
template <class T>
struct Stretch {
    const T* row;
    int begin, head, pieces, tail;
    __device__ __forceinline__ Stretch(const T* row_, int begin_, int end) : row(row_), begin(begin_) {
        constexpr int E = Elem<T>::E;
        const int off = (int)((reinterpret_cast<uintptr_t>(row + begin) / sizeof(T)) % E);
        head = min(end - begin, off ? E - off : 0);
        pieces = (end - begin - head) / E;
        tail = end - begin - head - pieces * E;
    }
    __device__ __forceinline__ const T* piece(int p) const { return row + begin + head + p * Elem<T>::E; }
    __device__ __forceinline__ int place(int p) const { return begin + head + p * Elem<T>::E; }
    // the single element of a thread, or -1: threads [0, E) the head's, [E, 2 E) the tail's
    __device__ __forceinline__ int single(int thread) const {
        constexpr int E = Elem<T>::E;
        if (thread < head) return begin + thread;
        if (thread >= E && thread < E + tail) return begin + head + pieces * E + thread - E;
        return -1;
    }
};

// m, s and t (in units of log2) of some elements
struct Sum { float m, s, t; };
__device__ __forceinline__ Sum join(Sum a, Sum b) {
    const float m = fmaxf(a.m, b.m);
    // differences of lowest and largest numbers overflow: at -2^20 the factor is 0 already
    const float da = fmaxf((a.m - m) * LOG2E, -0x1p20f), db = fmaxf((b.m - m) * LOG2E, -0x1p20f);
    const float ea = fast_exp2(da), eb = fast_exp2(db);
    return {m, a.s * ea + b.s * eb, (a.t + da * a.s) * ea + (b.t + db * b.s) * eb};
}
// N elements joined to a sum; the largest of them.  Where m is large the rounding of m log2(e) weighs more than a difference taken first: it is.
// An element of -infinity or near it makes t NaN, being 0 * infinity: the block is added once more, with bounded differences (a look at the
// least of the elements costs every block as much as a sixteenth of its exponentials).
template <bool ENTROPY, int N>
__device__ __forceinline__ float add(Sum& a, const float (&x)[N]) {
    float most = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) most = fmaxf(most, x[i]);
    if (most > a.m) {
        const float d = fmaxf((a.m - most) * LOG2E, -0x1p20f), e = fast_exp2(d);
        if constexpr (ENTROPY) a.t = (a.t + d * a.s) * e;
        a.s *= e;
        a.m = most;
    }
    // relative to c, which is m log2(e) but for its rounding: that much is put right for the sums
    const float c = a.m * LOG2E, off = -fmaf(a.m, LOG2E, -c), off_ln = off * LN2;
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float y = fmaf(x[i], LOG2E, -c), e = fast_exp2(y);
        s += e;
        if constexpr (ENTROPY) t = fmaf(y, e, t);
    }
    if constexpr (ENTROPY) t += fmaf(off, s, off_ln * t);
    s = fmaf(s, off_ln, s);
    const bool exact = fabsf(a.m) < TAME && (!ENTROPY || t == t);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!exact) != 0, 0) && !exact) {
        s = t = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float y = (x[i] - a.m) * LOG2E, e = fast_exp2(y);
            s += e;
            if constexpr (ENTROPY) t = fmaf(fmaxf(y, -0x1p20f), e, t);
        }
    }
    a.s += s;
    if constexpr (ENTROPY) a.t += t;
    return most;
}

// Elements in the order of the alternatives: larger first, equal ones by place; -0 is 0, and NaN the least.
__device__ __forceinline__ uint32_t order_of(float x) {           // of a number
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t rank_of(float x, uint32_t place) {
    return (uint64_t)order_of(x == x ? x : -__builtin_inff()) << 32 | (uint32_t)~place;
}
__device__ __forceinline__ float value_of(uint64_t rank) {
    const uint32_t b = (uint32_t)(rank >> 32);
    return __builtin_bit_cast(float, b >> 31 ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ uint32_t place_of(uint64_t rank) { return ~(uint32_t)rank; }

// A wave's, or a workgroup's, sums over its threads: the largest m first, then what the others come to beside it.
__device__ __forceinline__ Sum over_wave(Sum a) {
    const float m = row_ops::over_lanes<64>(a.m, row_ops::Max{});
    const float d = fmaxf((a.m - m) * LOG2E, -0x1p20f), e = fast_exp2(d);
    return {m, row_ops::over_lanes<64>(a.s * e, row_ops::Add{}), row_ops::over_lanes<64>((a.t + d * a.s) * e, row_ops::Add{})};
}

// What may still be among the alternatives.
struct Candidates {
    union {
        uint64_t list[LIST];
        uint16_t block[SLOTS][THREADS];       // of the largest of a thread's block, the upper half of its place in their order
    };
    uint64_t chosen[MAX_TOP];
    uint64_t best[WAVES];
    int count, blocks;
    float limit;
    uint16_t which[MOST_BLOCKS];              // the blocks that reach the limit: thread, and slot times THREADS
};
__device__ __forceinline__ uint64_t largest(uint64_t v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t w = __shfl_xor((unsigned long long)v, o, 64);
        v = w > v ? w : v;
    }
    return v;
}
// The top-th largest of a wave's N x 64 keys, or what it has of the bits from `least_bit` on, or a number between that and the next smaller
// key; 0 where there are fewer.
template <int N>
__device__ __forceinline__ uint32_t top_key(const uint32_t (&key)[N], int top, uint32_t least_bit) {
    uint32_t found = 0;
    for (uint32_t bit = 0x80000000u; bit >= least_bit && bit; bit >>= 1) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[k] >= (found | bit)));
        if (n >= top) found |= bit;
        if (n == top) break;
    }
    return found;
}
// c.chosen = the `top` largest of the first `count` of the list, in order, 0 behind the last; all threads call it.  A few by counting how many
// are larger than each; many, which are ties, by one search for each of the chosen.
__device__ __forceinline__ void choose(Candidates& c, int count, int top) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (count <= KEPT) {
        if ((int)threadIdx.x < top && (int)threadIdx.x >= count) c.chosen[threadIdx.x] = 0;
        for (int first = wave * 64; first < count; first += THREADS) {
            const bool has = first + lane < count;
            const uint64_t mine = has ? c.list[first + lane] : 0;
            int front = 0;
#pragma unroll 8
            for (int j = 0; j < count; ++j) front += c.list[j] > mine;
            if (has && front < top) c.chosen[front] = mine;
        }
    } else {
        uint64_t limit = ~(uint64_t)0;
        for (int j = 0; j < top; ++j) {
            uint64_t v = 0;
            for (int i = threadIdx.x; i < count; i += THREADS) {
                const uint64_t w = c.list[i];
                if (w < limit && w > v) v = w;
            }
            v = largest(v);
            if (lane == 0) c.best[wave] = v;
            __syncthreads();
            limit = c.best[0];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) limit = c.best[w] > limit ? c.best[w] : limit;
            if (threadIdx.x == 0) c.chosen[j] = limit;
            __syncthreads();
        }
    }
    __syncthreads();
}
// What one workgroup's stretch of a row comes to where rows are cut; its alternatives stand apart.
struct Part { float m, s, t, unused; };

struct Out {
    float *logp, *lse, *entropy, *top_logp;
    int32_t* top_ids;
};
// One thread writes a row's results, `top` threads its alternatives.
template <class T, bool ENTROPY>
__device__ __forceinline__ void write_row(const Out& out, size_t row, const T* x, int64_t target, int vocab, const Sum& a, float ls) {
    const bool none = a.s == 0.0f;                                // every logit is -infinity
    out.lse[row] = none ? -__builtin_inff() : a.m + ls;
    out.logp[row] = (uint64_t)target >= (uint64_t)vocab ? 0.0f : none ? -__builtin_inff() : (Elem<T>::one(x[target]) - a.m) - ls;
    if constexpr (ENTROPY) {
        const float h = ls - a.t * LN2 / a.s;
        out.entropy[row] = none || h < 0.0f ? 0.0f : h;
    }
}
__device__ __forceinline__ void write_top(const Out& out, size_t row, const Candidates& c, int top, const Sum& a, float ls) {
    const int j = threadIdx.x;
    if (j >= top) return;
    const uint64_t r = c.chosen[j];
    out.top_logp[row * top + j] = a.s == 0.0f ? -__builtin_inff() : (value_of(r) - a.m) - ls;
    out.top_ids[row * top + j] = (int32_t)place_of(r);
}
__device__ __forceinline__ int64_t target_of(const void* targets, int is64, size_t row) {
    return is64 ? static_cast<const int64_t*>(targets)[row] : static_cast<const int32_t*>(targets)[row];
}
}  // namespace lp

// Workgroup (row, part of it).  Rows of one part are finished here, others leave a Part and their alternatives.  A pass over 4096 x 50001 bf16
// with entropy and 5 alternatives 75 us, 5.5 TB/s; 32 x 131072 with 20 8.6 us, 4.3 of them without alternatives.
template <class T, bool CACHED, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(lp::THREADS) void token_logprobs_kernel(const T* __restrict__ logits, const void* __restrict__ targets, int targets64,
                                                                     lp::Out out, lp::Part* __restrict__ parts, uint64_t* __restrict__ part_tops,
                                                                     int vocab, size_t width, int cut, int each, int top) {
    using namespace lp;
    constexpr int E = Elem<T>::E;
    __shared__ Sum sums[WAVES];
    const size_t row = blockIdx.x / cut;
    const int part = blockIdx.x % cut, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* x = logits + row * width;
    const int begin = min(vocab, part * each), end = min(vocab, begin + each);
    const Stretch<T> st(x, begin, end);
    Sum a{LEAST, 0.0f, 0.0f};
    const int alone = st.single(threadIdx.x);
    const float single[1] = {alone >= 0 ? Elem<T>::one(x[alone]) : -__builtin_inff()};
    __shared__ typename std::conditional<TOP, float[THREADS], float[1]>::type most;
    __shared__ typename std::conditional<TOP, Candidates, char>::type c;
    int blocks = 0;
    // the maximum of the next block; a thread reads no other's
    auto keep = [&](float m) {
        if constexpr (TOP) {
            uint16_t* at = &c.block[blocks % SLOTS][threadIdx.x];
            const uint16_t now = (uint16_t)(order_of(m) >> 16);
            *at = blocks < SLOTS ? now : max(now, *at);
            ++blocks;
        }
    };
    int p = threadIdx.x;
    for (; p + (AT_ONCE - 1) * THREADS < st.pieces; p += AT_ONCE * THREADS) {
        u32x4 v[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) v[u] = ld_stream_16<CACHED>(st.piece(p + u * THREADS));
        float f[AT_ONCE * E];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            float g[E];
            Elem<T>::unpack(v[u], g);
#pragma unroll
            for (int i = 0; i < E; ++i) f[u * E + i] = g[i];
        }
        keep(add<ENTROPY>(a, f));
    }
    if (p < st.pieces) {
        float m = LEAST;
        for (; p < st.pieces; p += THREADS) {
            float f[E];
            Elem<T>::unpack(ld_stream_16<CACHED>(st.piece(p)), f);
            m = fmaxf(m, add<ENTROPY>(a, f));
        }
        keep(m);
    }
    if (alone >= 0) add<ENTROPY>(a, single);
    const float mine = a.m;                                       // the largest of this thread's elements
    a = over_wave(a);
    if (lane == 0) sums[wave] = a;
    if constexpr (TOP) {
        most[threadIdx.x] = mine;
        if (threadIdx.x == 0) c.count = c.blocks = 0;
    }
    __syncthreads();
    a = sums[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) a = join(a, sums[w]);
    const float ls = logf(a.s);
    if (threadIdx.x == 0) {
        if (cut > 1) parts[blockIdx.x] = Part{a.m, a.s, a.t, 0.0f};
        else write_row<T, ENTROPY>(out, row, x, target_of(targets, targets64, row), vocab, a, ls);
    }
    if constexpr (TOP) {
        // No element below the top-th largest of the threads' largest is an alternative; nor below that of four threads' together, which is one
        // key a lane and for small `top` hardly less.  One wave looks for it, by the upper 16 bits of the keys.  One key a lane is faster for few rows
        // (32 x 131072, top 8 13.9 us and by four 14.6, 20 15.7 and 16.4, 28 16.6 and 17.1), and slower for many from some 28 alternatives on, the
        // more so the nearer they are to the 64 keys (4096 x 50001, 28 82.3 and 81.5, 48 94.1 and 86.1, 64 613 and 91).
        if (wave == 0) {
            uint32_t key[WAVES], four[1] = {0};
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                key[w] = order_of(most[w * 64 + lane]);
                four[0] = max(four[0], key[w]);
            }
            const float found = value_of((uint64_t)(top <= 24 ? top_key(four, top, 0x10000u) : top_key(key, top, 0x10000u)) << 32);
            // none where fewer than `top` threads have elements that are numbers
            if (lane == 0) c.limit = found > LEAST ? found : -__builtin_inff();
        }
        __syncthreads();
        const float limit = c.limit;
        const bool all = limit == -__builtin_inff();
        if (all || mine >= limit) {
            const uint32_t least = all ? 0 : order_of(limit) >> 16;
            for (int k = 0; k < min(blocks, SLOTS); ++k)
                if (c.block[k][threadIdx.x] >= least) {
                    const int at = atomicAdd(&c.blocks, 1);
                    if (at < MOST_BLOCKS) c.which[at] = (uint16_t)(k * THREADS + threadIdx.x);
                }
        }
        __syncthreads();
        // elements of a piece go to the list, those that reach the limit and are above `least`
        auto offer = [&](int piece, uint64_t least) {
            if (piece >= st.pieces) return;
            float f[E];
            Elem<T>::unpack(ld_global_16(st.piece(piece)), f);
            const int place = st.place(piece);
            uint32_t mine = 0;                                    // a bit for each
#pragma unroll
            for (int i = 0; i < E; ++i)
                if ((all || f[i] >= limit) && (least == 0 || rank_of(f[i], place + i) > least)) mine |= 1u << i;
            if (!mine) return;
            int at = atomicAdd(&c.count, __builtin_popcount(mine));
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (mine >> i & 1) {
                    if (at < LIST) c.list[at] = rank_of(f[i], place + i);
                    ++at;
                }
        };
        auto offer_single = [&](uint64_t least) {
            if (alone < 0 || !(all || single[0] >= limit) || rank_of(single[0], alone) <= least) return;
            const int at = atomicAdd(&c.count, 1);
            if (at < LIST) c.list[at] = rank_of(single[0], alone);
        };
        // the blocks that reach the limit, a piece a thread
        const int found = c.blocks;
        if (found <= MOST_BLOCKS) {
            for (int i = threadIdx.x; i < found * AT_ONCE; i += THREADS) {
                const int which = c.which[i / AT_ONCE];
                for (int p = which % THREADS + (which / THREADS * AT_ONCE + i % AT_ONCE) * THREADS; p < st.pieces; p += SLOTS * AT_ONCE * THREADS) offer(p, 0);
            }
            offer_single(0);
        }
        __syncthreads();
        int count = c.count;
        if (count > LIST || found > MOST_BLOCKS) {
            // Many are as large: all elements once more, TURN threads' pieces in a turn, and whenever there are many the first of them go on.
            __syncthreads();
            if (threadIdx.x == 0) c.count = 0;
            __syncthreads();
            const int turns = (st.pieces + TURN - 1) / TURN;
            uint64_t least = 0;
            for (int turn = 0; turn <= turns; ++turn) {
                if (turn < turns) {
                    if (threadIdx.x < TURN) offer(turn * TURN + threadIdx.x, least);
                } else {
                    offer_single(least);
                }
                __syncthreads();
                count = c.count;
                __syncthreads();
                if (turn < turns && count > KEPT) {
                    choose(c, count, top);
                    least = c.chosen[top - 1];
                    if (threadIdx.x < top) c.list[threadIdx.x] = c.chosen[threadIdx.x];
                    if (threadIdx.x == 0) c.count = top;
                    __syncthreads();
                }
            }
        }
        choose(c, count, top);
        if (cut > 1) {
            // the first of all parts, then the second, ...
            if (threadIdx.x < top) part_tops[(row * top + threadIdx.x) * cut + part] = c.chosen[threadIdx.x];
        } else {
            write_top(out, row, c, top, a, ls);
        }
    }
}

// Rows that were cut: a workgroup a row.  32 rows of 32 parts with 20 alternatives 4.5 us.
template <class T, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(lp::THREADS) void token_logprobs_join_kernel(const T* __restrict__ logits, const void* __restrict__ targets, int targets64,
                                                                          lp::Out out, const lp::Part* __restrict__ parts,
                                                                          const uint64_t* __restrict__ part_tops, int vocab, size_t width, int cut, int top) {
    using namespace lp;
    const size_t row = blockIdx.x;
    const int lane = threadIdx.x & 63;
    const T* x = logits + row * width;
    Sum a{LEAST, 0.0f, 0.0f};
    for (int i = lane; i < cut; i += 64) {                        // every wave by itself
        const Part q = parts[row * cut + i];
        a = join(a, Sum{q.m, q.s, q.t});
    }
    // No alternative is below the top-th largest of each part's first few: one key a lane, or four.  128 and fewer are all put
    // in order (160 12.1 us with a limit, 12.4 without; 32 12.9 and 11.4).  One key a lane where that is two of each part or more and `top` is far
    // below 64: 32 x 131072 of 32 parts, top 16 14.9 us so and 15.1 by four, 20 15.6 and 15.9, 24 15.8 and 16.0.
    constexpr uint32_t LEAST_BIT = sizeof(T) == 2 ? 0x10000 : 1;
    const bool all = cut * top <= THREADS / 2;
    uint32_t limit = 0;
    uint64_t mine = 0;
    if constexpr (TOP) {
        const uint64_t* ranks = part_tops + row * cut * top;
        auto key_of = [&](int i, int first) { return i < cut * first ? (uint32_t)(ranks[i] >> 32) : 0; };
        if (all) {
            if ((int)threadIdx.x < cut * top) mine = ranks[threadIdx.x];
        } else if (top <= 24 && cut <= 32) {
            const uint32_t key[1] = {key_of(lane, min(top, 64 / cut))};
            limit = top_key(key, top, LEAST_BIT);
        } else {
            uint32_t key[JOINED / 64];
#pragma unroll
            for (int k = 0; k < JOINED / 64; ++k) key[k] = key_of(lane + 64 * k, min(top, JOINED / cut));
            limit = top_key(key, top, LEAST_BIT);
        }
    }
    a = over_wave(a);
    const float ls = logf(a.s);
    if (threadIdx.x == 0) write_row<T, ENTROPY>(out, row, x, target_of(targets, targets64, row), vocab, a, ls);
    if constexpr (TOP) {
        __shared__ Candidates c;
        if (threadIdx.x == 0) c.count = 0;
        __syncthreads();
        if (all) {
            c.list[threadIdx.x] = mine;                           // 0, no element, is behind all of them
        } else {
            for (int i = threadIdx.x; i < cut * top; i += THREADS) {  // at most as many as the list holds
                const uint64_t r = part_tops[row * cut * top + i];
                if (r != 0 && (uint32_t)(r >> 32) >= limit) c.list[atomicAdd(&c.count, 1)] = r;
            }
        }
        __syncthreads();
        choose(c, all ? cut * top : c.count, top);
        write_top(out, row, c, top, a, ls);
    }
}

// The gradient: workgroup (row, part of it).  logits and d_logits may be the same memory: a thread writes where it alone has read.  A pass
// over 4096 x 50001 bf16 130 us, 6.3 TB/s; 777 x 50001 f32 with entropy 52.7, 5.9 TB/s.
template <class T, bool CACHED, bool ENTROPY>
__global__ __launch_bounds__(lp::BWD_THREADS) void token_logprobs_bwd_kernel(const T* logits, const void* __restrict__ targets, int targets64,
                                                                         const float* __restrict__ lse, const float* __restrict__ entropy,
                                                                         const float* __restrict__ d_logp, const float* __restrict__ d_entropy,
                                                                         const float* __restrict__ d_lse, T* d_logits, int vocab, size_t width,
                                                                         int cut, int each) {
    using namespace lp;
    constexpr int E = Elem<T>::E;
    const size_t row = blockIdx.x / cut;
    const int part = blockIdx.x % cut;
    const T* x = logits + row * width;
    T* dx = d_logits + row * width;
    const int begin = min(vocab, part * each), end = min(vocab, begin + each);
    const Stretch<T> st(x, begin, end);
    const int64_t given = target_of(targets, targets64, row);
    const bool has_target = (uint64_t)given < (uint64_t)vocab && d_logp;
    const int target = has_target ? (int)given : -1;
    const float g = has_target ? d_logp[row] : 0.0f, gh = ENTROPY ? d_entropy[row] : 0.0f, l = lse[row];
    float k = (d_lse ? d_lse[row] : 0.0f) - g, kh = -gh * LN2;    // dx = p (k + kh log2 p)
    // a row without a gradient, or without a logit above -infinity
    const bool zero = (g == 0.0f && k == 0.0f && gh == 0.0f) || l == -__builtin_inff();
    if constexpr (ENTROPY) k -= gh != 0.0f ? gh * entropy[row] : 0.0f;      // an entropy without a gradient may be NaN
    // dx = e (k + kh y) with e = 2^y; y is relative to c, which is lse log2(e) but for its rounding: that much goes into k and kh
    const bool tame = fabsf(l) < 0x1p20f;
    const float c = l * LOG2E;
    if (tame) {
        const float off = -fmaf(l, LOG2E, -c), e = fast_exp2(off);
        k = fmaf(kh, off, k) * e;
        kh *= e;
    }
    auto slope = [&](float v) {
        const float y = tame ? fmaf(v, LOG2E, -c) : (v - l) * LOG2E;
        const float e = fast_exp2(y);
        if constexpr (ENTROPY) return e * fmaf(fmaxf(y, -0x1p20f), kh, k);
        else return e * k;
    };
    auto with_target = [&](float v, bool there) {                 // the same bits wherever an element is computed
#pragma clang fp contract(off)
        return there ? v + g : v;
    };
    auto put = [&](int i) { Elem<T>::put(dx + i, zero ? 0.0f : with_target(slope(Elem<T>::one(x[i])), i == target)); };
    // pieces of 16 bytes where both tensors have them at the same elements
    if ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(d_logits)) % 16 != 0) {
        for (int i = begin + threadIdx.x; i < end; i += BWD_THREADS) put(i);
    } else {
        const int alone = st.single(threadIdx.x);
        if (alone >= 0) put(alone);
        for (int p0 = threadIdx.x; p0 < st.pieces; p0 += BWD_AT_ONCE * BWD_THREADS) {
            u32x4 v[BWD_AT_ONCE];
            if (!zero) {
#pragma unroll
                for (int u = 0; u < BWD_AT_ONCE; ++u) v[u] = ld_stream_16<CACHED>(st.piece(min(p0 + u * BWD_THREADS, st.pieces - 1)));
            }
#pragma unroll
            for (int u = 0; u < BWD_AT_ONCE; ++u) {
                const int p = p0 + u * BWD_THREADS;
                if (p >= st.pieces) break;
                float f[E];
                if (zero) {
#pragma unroll
                    for (int i = 0; i < E; ++i) f[i] = 0.0f;
                } else {
                    Elem<T>::unpack(v[u], f);
#pragma unroll
                    for (int i = 0; i < E; ++i) f[i] = slope(f[i]);
                    const int at = target - st.place(p);
                    if ((unsigned)at < (unsigned)E) {
#pragma unroll
                        for (int i = 0; i < E; ++i) f[i] = with_target(f[i], i == at);
                    }
                }
                st_global_16_nt(dx + st.place(p), Elem<T>::pack(f));
            }
        }
    }
    if (part == cut - 1)
        for (size_t i = vocab + threadIdx.x; i < width; i += BWD_THREADS) Elem<T>::put(dx + i, 0.0f);
}

// ------------------------------------------------------------------------------------------
namespace {
using namespace lp;
// Parts of a row, so that few rows fill the device: up to 1024 workgroups of 8 KB of a row or more; what the parts leave for the alternatives fits
// the list that joins them.
struct Cut { int parts, each; };
Cut cut_of(size_t rows, int vocab, int elem_bytes, int top) {
    size_t n = std::min((size_t)1024 / rows, (size_t)JOINED / 2);
    n = std::min(n, (size_t)vocab * elem_bytes / 8192);
    if (top) n = std::min(n, (size_t)LIST / top);
    n = std::max(n, (size_t)1);
    const int each = (int)(((vocab + n - 1) / n + 127) / 128 * 128);
    return {(vocab + each - 1) / each, each};
}
// of the gradient: a workgroup's threads go round once
int bwd_each(int elem_bytes) { return BWD_THREADS * BWD_AT_ONCE * 16 / elem_bytes; }
}  // namespace

bool token_logprobs_fits(size_t rows, int vocab, int bf16) {
    const int each = bwd_each(bf16 ? 2 : 4);
    return rows < ((size_t)1 << 24) && rows * ((vocab + each - 1) / each) < ((size_t)1 << 24);      // workgroups of 256 threads
}

size_t token_logprobs_workspace_bytes(size_t rows, int vocab, int top, int bf16) {
    const Cut c = cut_of(rows, vocab, bf16 ? 2 : 4, top);
    return c.parts > 1 ? rows * c.parts * (sizeof(Part) + 8 * (size_t)top) : 0;
}

int launch_token_logprobs(const void* logits, const void* targets, int targets64, float* logp, float* lse, float* entropy, float* top_logp,
                          int32_t* top_ids, size_t rows, int vocab, size_t width, int top, int bf16, void* workspace, hipStream_t stream) {
    const Cut c = cut_of(rows, vocab, bf16 ? 2 : 4, top);
    const Out out{logp, lse, entropy, top_logp, top_ids};
    Part* parts = static_cast<Part*>(workspace);
    uint64_t* tops = reinterpret_cast<uint64_t*>(parts + (c.parts > 1 ? rows * c.parts : 0));
    const bool cached = rows * vocab * (bf16 ? 2 : 4) <= kStreamCached;
    auto go = [&](auto elem, auto in_cache, auto with_entropy, auto with_top) {
        using T = decltype(elem);
        const T* x = static_cast<const T*>(logits);
        launch_kernel((token_logprobs_kernel<T, in_cache(), with_entropy(), with_top()>), dim3((unsigned)(rows * c.parts)), dim3(THREADS), 0, stream, x,
                      targets, targets64, out, parts, tops, vocab, width, c.parts, c.each, top);
        if (c.parts > 1)
            launch_kernel((token_logprobs_join_kernel<T, with_entropy(), with_top()>), dim3((unsigned)rows), dim3(THREADS), 0, stream, x, targets, targets64,
                          out, parts, tops, vocab, width, c.parts, top);
    };
    auto outputs = [&](auto elem, auto in_cache) {
        if (entropy) { if (top) go(elem, in_cache, std::true_type{}, std::true_type{}); else go(elem, in_cache, std::true_type{}, std::false_type{}); }
        else { if (top) go(elem, in_cache, std::false_type{}, std::true_type{}); else go(elem, in_cache, std::false_type{}, std::false_type{}); }
    };
    auto pick = [&](auto elem) { if (cached) outputs(elem, std::true_type{}); else outputs(elem, std::false_type{}); };
    if (bf16) pick(uint16_t{}); else pick(float{});
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

int launch_token_logprobs_bwd(const void* logits, const void* targets, int targets64, const float* lse, const float* entropy, const float* d_logp,
                              const float* d_entropy, const float* d_lse, void* d_logits, size_t rows, int vocab, size_t width, int bf16,
                              hipStream_t stream) {
    const int most = bwd_each(bf16 ? 2 : 4), cut = (vocab + most - 1) / most;
    const int each = ((vocab + cut - 1) / cut + 63) / 64 * 64;       // of equal parts, at most `most`
    const bool cached = rows * vocab * (bf16 ? 4 : 8) <= kStreamCached;
    auto go = [&](auto elem, auto in_cache, auto with_entropy) {
        using T = decltype(elem);
        launch_kernel((token_logprobs_bwd_kernel<T, in_cache(), with_entropy()>), dim3((unsigned)(rows * cut)), dim3(BWD_THREADS), 0, stream,
                      static_cast<const T*>(logits), targets, targets64, lse, entropy, d_logp, d_entropy, d_lse, static_cast<T*>(d_logits), vocab, width, cut,
                      each);
    };
    auto pick = [&](auto elem) {
        if (cached) { if (d_entropy) go(elem, std::true_type{}, std::true_type{}); else go(elem, std::true_type{}, std::false_type{}); }
        else { if (d_entropy) go(elem, std::false_type{}, std::true_type{}); else go(elem, std::false_type{}, std::false_type{}); }
    };
    if (bf16) pick(uint16_t{}); else pick(float{});
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tyr
