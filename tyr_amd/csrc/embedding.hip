// Embedding: rows of a table by token, and the gradient of the table (gfx950).
//
//   out[i] = scale table[ids[i]]                          a token outside of the table (padding) gives a row of zeros
//   G[v]   = scale sum over i with ids[i] = v of d_out[i]  (or that added to a gradient that is there); such a token adds nothing
//
// The gradient is summed by sorted tokens: no atomic additions of floating point, the same bits every time.  Three ways:
//   few tokens       one launch: a workgroup has the tokens of its residue class, finds them among all, adds their rows, and clears the others
//   up to 24576      such classes put their pairs (token, place) together, equal tokens side by side; then the sums
//   more             a radix sort of the pairs, then the sums
// The sort notes which tokens are there, and beside the sums the rows of the others are cleared.  The sort's own launches leave the memory idle:
// beside them the end of the table is cleared as a whole, where tokens are rare if they are numbered by how frequent they are.
// The sums: a wave adds the rows of PIECE consecutive pairs, 16 bytes of a row a lane, in f32.  A run of equal tokens no longer than that belongs to
// the wave of the piece that it begins in; a longer one leaves an f32 row for each piece that it reaches into, and a last launch adds those.
//
// Bound by HBM: the lookup reads and writes its rows, the gradient reads d_out and writes the table once (zeros for the tokens that are not
// there), or reads and writes the tokens' rows only.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "common.hpp"
#include "launch.hpp"

namespace tyr {

namespace emb {
// a row as 16-byte pieces of E elements
template <class T> struct Row;
template <> struct Row<uint16_t> {
    static constexpr int E = 8;
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = bf16_lo(v[i]); f[2 * i + 1] = bf16_hi(v[i]); }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
        return u32x4{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])};
    }
};
template <> struct Row<float> {
    static constexpr int E = 4;
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[4]) {
        const f32x4 x = __builtin_bit_cast(f32x4, v);              // (a bit cast of one element of a vector reads the first)
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = x[i];
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[4]) {
        return __builtin_bit_cast(u32x4, f32x4{f[0], f[1], f[2], f[3]});
    }
};
// A token as the sort sees it: those of the table below 2^31, the others above.
__device__ __forceinline__ uint32_t key_of(int32_t id) { return (uint32_t)id; }
__device__ __forceinline__ uint32_t key_of(int64_t id) { return (uint64_t)id >> 31 ? 0xffffffffu : (uint32_t)id; }

constexpr int CLASSES = 256;              // residue classes of tokens, a workgroup each
// Tokens times 64-lane blocks of a row, of one launch.  900 tokens of 1024 bf16 15.1 us so (half of them one token 24.6) and 20.6 (21.9) as the next
// form; 1800 17.7 (35.2) so and 20.9 (23.4).
constexpr int FEW = 2048;
// Tokens at most that classes put together.  20000 28.8 us so (half of them one token 50.3) and 36.1 (48.5) by the radix sort; 30000 34.5 (67.0), 41.8 (57.8).
constexpr int GATHERED = 3 << 13;
constexpr int MAX_QUOTIENTS = 1024;       // quotients by CLASSES at most, for both
constexpr int CHUNK = 1024, CHUNKS = 128; // radix sort: tokens of a turn, workgroups at most
constexpr int MAX_DIGIT = 9;
constexpr int CLEARED = 16;               // 16-byte pieces that a thread of 1024 fills with zeros
// Bytes of the table cleared beside the classes, beside a launch of the radix sort.  24500 tokens of a 65536 x 2048 bf16 table 74 us, without 80;
// 32768 89.0, with 20 MB 91.0, without 100.
constexpr size_t BESIDE = (size_t)48 << 20, BESIDE_PASS = (size_t)32 << 20;
constexpr int HELD = 256;                 // pairs that a wave keeps of its share
}  // namespace emb

// 2^shift threads a row, 256 >> shift rows a workgroup.  16384 rows of 65536 x 2048 bf16 16.3 us: 67 MB written past the caches and 26 MB of
// distinct rows read, 5.7 TB/s.
template <class T, class I>
__global__ __launch_bounds__(256) void embedding_kernel(const I* __restrict__ ids, const T* __restrict__ table, T* __restrict__ out, size_t n,
                                                        uint32_t vocab, int pieces, int shift, float scale) {
    using R = emb::Row<T>;
    const size_t token = (size_t)blockIdx.x * (256 >> shift) + (threadIdx.x >> shift);
    if (token >= n) return;
    const uint32_t id = emb::key_of(ids[token]);
    const T* from = table + (size_t)id * pieces * R::E;
    T* to = out + token * pieces * R::E;
    for (int p = threadIdx.x & ((1 << shift) - 1); p < pieces; p += 1 << shift) {
        u32x4 v = {0, 0, 0, 0};
        if (id < vocab) {
            float f[R::E];
            R::unpack(ld_global_16(from + p * R::E), f);
#pragma unroll
            for (int i = 0; i < R::E; ++i) f[i] *= scale;
            v = R::pack(f);
        }
        st_global_16_nt(to + p * R::E, v);
    }
}

// ---- the sort

// A row of zeros by one wave.
template <class T>
__device__ __forceinline__ void clear_row(T* row, int row_pieces) {
    for (int p = threadIdx.x & 63; p < row_pieces; p += 64) st_global_16_nt(row + p * emb::Row<T>::E, u32x4{0, 0, 0, 0});
}
// Zeros: `pieces` of 16 bytes, their share of workgroup w of 1024 threads.
struct Zeros {
    void* at;
    size_t pieces;
    __device__ __forceinline__ void fill(uint32_t w) const {
        const size_t first = (size_t)w * (1024 * emb::CLEARED) + threadIdx.x;
#pragma unroll
        for (int k = 0; k < emb::CLEARED; ++k)
            if (first + k * 1024 < pieces) st_global_16_nt(static_cast<char*>(at) + (first + k * 1024) * 16, u32x4{0, 0, 0, 0});
    }
    __host__ uint32_t workgroups() const { return (uint32_t)((pieces + 1024 * emb::CLEARED - 1) / (1024 * emb::CLEARED)); }
};
// f32 sums to a row of the table, or with what is there of it
template <class T, bool INTO>
__device__ __forceinline__ void finish(T* to, float (&sum)[emb::Row<T>::E], float scale, u32x4 there) {
    using R = emb::Row<T>;
#pragma unroll
    for (int i = 0; i < R::E; ++i) sum[i] *= scale;
    if constexpr (INTO) {
        float old[R::E];
        R::unpack(there, old);
#pragma unroll
        for (int i = 0; i < R::E; ++i) sum[i] += old[i];
    }
    st_global_16_nt(to, R::pack(sum));
}
template <class T>
__device__ __forceinline__ void finish(T* to, float (&sum)[emb::Row<T>::E], float scale, bool into) {
    if (into) finish<T, true>(to, sum, scale, ld_global_16(to)); else finish<T, false>(to, sum, scale, u32x4{});
}
// Lanes in front that are set.
__device__ __forceinline__ int before(uint64_t lanes) { return __builtin_popcountll(lanes & (((uint64_t)1 << (threadIdx.x & 63)) - 1)); }

// One chunk of up to 1024 items, one a thread, in their order: place[digit] goes on by how many there are of it; the item's own place is the
// result.  16 waves; `count` is 0 before and after.  Ends with a barrier.
template <int DIGITS>
__device__ __forceinline__ uint32_t take_places(uint32_t (&place)[DIGITS], uint16_t (&count)[16][DIGITS], uint32_t digit, bool real, int bits) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint64_t same = __builtin_amdgcn_ballot_w64(real);
    for (int b = 0; b < bits; ++b) {
        const uint64_t set = __builtin_amdgcn_ballot_w64(digit >> b & 1);
        same &= digit >> b & 1 ? set : ~set;
    }
    const int rank = before(same);
    const bool leads = real && rank == 0;
    if (leads) count[wave][digit] = (uint16_t)__builtin_popcountll(same);
    __syncthreads();
    uint32_t to = place[digit] + rank;
#pragma unroll 4
    for (int w = 0; w < wave; ++w) to += count[w][digit];
    __syncthreads();
    if (leads) {
        atomicAdd(&place[digit], (uint32_t)__builtin_popcountll(same));
        count[wave][digit] = 0;
    }
    __syncthreads();
    return to;
}
// place[d] += the sum of total[0, d), by one wave; digits a power of two
__device__ __forceinline__ void add_scan(uint32_t* place, const uint32_t* total, int digits) {
    const int lane = threadIdx.x & 63, each = max(1, digits / 64), d0 = lane * each;
    uint32_t sum = 0;
    if (d0 < digits)
        for (int k = 0; k < each; ++k) sum += total[d0 + k];
    uint32_t front = sum;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t other = __shfl_up(front, o, 64);
        if (lane >= o) front += other;
    }
    front -= sum;
    if (d0 < digits)
        for (int k = 0; k < each; ++k) {
            place[d0 + k] += front;
            front += total[d0 + k];
        }
}

// Classes: workgroup c has the tokens that are c modulo CLASSES.  It counts over all ids how many pairs stand in front of its own, those of
// smaller classes, and how many each wave finds of each quotient in its share of the ids; so every wave knows where its pairs go and puts them
// there without another's help.  there[token] = whether it is.  Workgroups behind the classes clear the end of the table.  LDS:
// count [16][digits], total and front [digits].  16384 tokens 9.1 us, which is latency: ids, counts, a scan.
template <class I>
__global__ __launch_bounds__(1024, 8) void embedding_gather_kernel(const I* __restrict__ ids, u32x2* __restrict__ pairs, uint8_t* __restrict__ there, int n,
                                                                   uint32_t vocab, int bits, Zeros zeros) {
    using namespace emb;
    __shared__ u32x2 held[16][HELD];
    __shared__ int mine_of[16], front_of[16];
    extern __shared__ __attribute__((aligned(16))) uint32_t total[];
    if (blockIdx.x >= CLASSES) return zeros.fill(blockIdx.x - CLASSES);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), digits = 1 << bits;
    uint32_t* const place = total + digits;
    uint32_t* const counts = place + digits;                        // of wave w, two quotients a word
    uint16_t* const count = reinterpret_cast<uint16_t*>(counts) + (wave << bits);
    const uint32_t c = blockIdx.x;
    for (int d = threadIdx.x; d < digits; d += 1024) place[d] = 0;
    for (int d = threadIdx.x; d < 8 * digits; d += 1024) counts[d] = 0;
    __syncthreads();
    const int share = ((n + 15) / 16 + 63) / 64 * 64, first = wave * share, end = min(n, first + share);
    int mine = 0, front = 0;
    // the share's ids, AHEAD x 64 asked for together; `take` gets 64 pairs at a time, those of this class marked
    constexpr int AHEAD = 8;
    auto look = [&](auto take) {
        for (int i0 = first; i0 < end; i0 += 64 * AHEAD) {
            I id[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) id[u] = ids[min(i0 + 64 * u + lane, n - 1)];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int i = i0 + 64 * u + lane;
                const uint32_t key = i < end ? key_of(id[u]) : 0xffffffffu;
                take(u32x2{key, (uint32_t)i}, key < vocab && key % CLASSES == c);
            }
        }
    };
    look([&](u32x2 pair, bool own) {
        front += __builtin_popcountll(__builtin_amdgcn_ballot_w64(pair.x < vocab && pair.x % CLASSES < c));
        const uint64_t them = __builtin_amdgcn_ballot_w64(own);
        if (!them) return;
        if (own) {
            const int k = mine + before(them);
            if (k < HELD) held[wave][k] = pair;
            const uint32_t d = (wave << bits) + pair.x / CLASSES;
            atomicAdd(&counts[d >> 1], d & 1 ? 0x10000u : 1u);
        }
        mine += __builtin_popcountll(them);
    });
    if (lane == 0) {
        mine_of[wave] = mine;
        front_of[wave] = front;
    }
    __syncthreads();
    int all_mine = 0, all_front = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        all_mine += mine_of[w];
        all_front += front_of[w];
    }
    // of a quotient: all of it, and in the place of each wave's count what the waves in front have
    for (int d = threadIdx.x; d < digits; d += 1024) {
        uint16_t* of = reinterpret_cast<uint16_t*>(counts) + d;
        uint32_t sum = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const uint32_t k = of[w << bits];
            of[w << bits] = (uint16_t)sum;
            sum += k;
        }
        total[d] = sum;
        if (d * CLASSES + c < vocab) there[d * CLASSES + c] = sum != 0;
    }
    // places of no pair, behind the last
    if (c == CLASSES - 1)
        for (int i = all_front + all_mine + threadIdx.x; i < n; i += 1024) pairs[i] = u32x2{0xffffffffu, 0};
    __syncthreads();
    if (wave == 0) add_scan(place, total, digits);
    __syncthreads();
    auto put = [&](u32x2 pair, bool own) {
        uint64_t same = __builtin_amdgcn_ballot_w64(own);
        if (!same) return;
        const uint32_t d = own ? pair.x / CLASSES : 0, first = __builtin_amdgcn_readlane(d, __builtin_ctzll(same));
        if (__builtin_amdgcn_ballot_w64(own && d != first))
            for (int b = 0; b < bits; ++b) {
                const uint64_t set = __builtin_amdgcn_ballot_w64(d >> b & 1);
                same &= d >> b & 1 ? set : ~set;
            }
        const int rank = before(same);
        const uint32_t at = count[d];
        if (own) {
            pairs[all_front + place[d] + at + rank] = pair;
            if (rank == 0) count[d] = (uint16_t)(at + __builtin_popcountll(same));
        }
    };
    if (mine > HELD) look(put);
    else
        for (int k = 0; k < mine; k += 64) {
            const bool own = k + lane < mine;
            put(own ? held[wave][k + lane] : u32x2{0, 0}, own);
        }
}

// Few tokens, all in one launch.  A workgroup keeps its class's pairs in LDS and clears the rows of the others.  Tokens that are there up to
// LIGHT times are summed by one group of waves that covers a row; more frequent ones by all groups, joined through LDS.  900 tokens of a
// 32768 x 1024 bf16 table 13.9 us, 67 MB of them zeros: 4.9 TB/s with 3 us of looking for the tokens.
template <class T, class I>
__global__ __launch_bounds__(1024) void embedding_few_kernel(const I* __restrict__ ids, const T* __restrict__ d_out, T* __restrict__ table, int n,
                                                             uint32_t vocab, int row_pieces, int blocks, float scale, bool into) {
    using namespace emb;
    using R = Row<T>;
    constexpr int E = R::E, LIGHT = 8;
    __shared__ uint32_t keys[FEW], places[FEW];                    // of the class, in order
    __shared__ uint32_t count[MAX_QUOTIENTS];                      // of a quotient
    __shared__ uint16_t light[MAX_QUOTIENTS], heavy[MAX_QUOTIENTS];
    __shared__ uint32_t few_rows[16][LIGHT], many_rows[FEW];
    __shared__ int own_of[16], lights, heavies;
    __shared__ f32x4 sums[16][E / 4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t c = blockIdx.x;
    if (c >= vocab) return;
    const int quotients = (int)((vocab - 1 - c) / CLASSES + 1);
    if (threadIdx.x == 0) lights = heavies = 0;
    if ((int)threadIdx.x < quotients) count[threadIdx.x] = 0;
    int m = 0;
    for (int i0 = 0; i0 < n; i0 += 1024) {
        const int i = i0 + threadIdx.x;
        const uint32_t key = i < n ? key_of(ids[i]) : 0xffffffffu;
        const bool own = key < vocab && key % CLASSES == c;
        const uint64_t them = __builtin_amdgcn_ballot_w64(own);
        if (lane == 0) own_of[wave] = __builtin_popcountll(them);
        __syncthreads();
        int at = m;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            at += w < wave ? own_of[w] : 0;
            m += own_of[w];
        }
        if (own) {
            keys[at + before(them)] = key;
            places[at + before(them)] = (uint32_t)i;
            atomicAdd(&count[key / CLASSES], 1u);
        }
        __syncthreads();
    }
    if ((int)threadIdx.x < quotients && count[threadIdx.x] != 0) {
        if (count[threadIdx.x] <= LIGHT) light[atomicAdd(&lights, 1)] = (uint16_t)threadIdx.x;
        else heavy[atomicAdd(&heavies, 1)] = (uint16_t)threadIdx.x;
    }
    __syncthreads();
    const size_t d = (size_t)row_pieces * E;
    // waves side by side cover `across` blocks of a row; so many groups of them
    const int across = min(blocks, 16), groups = 16 / across, group = wave / across, first_block = wave % across;
    // the sum of rows[from], rows[from + step], ... of them in d_out
    auto add_rows = [&](const uint32_t* rows, int count, int from, int step, int block, float (&sum)[E]) {
        constexpr int AHEAD = 8;
        const T* at = d_out + min(block * 64 + lane, row_pieces - 1) * E;
#pragma unroll
        for (int i = 0; i < E; ++i) sum[i] = 0.0f;
        for (int r = from; r < count; r += step * AHEAD) {
            u32x4 row[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) row[u] = ld_global_16(at + (size_t)__builtin_amdgcn_readfirstlane(rows[min(r + u * step, count - 1)]) * d);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {                     // without a branch, behind which the loads would wait for each other
                float f[E];
                R::unpack(r + u * step < count ? row[u] : u32x4{0, 0, 0, 0}, f);
#pragma unroll
                for (int i = 0; i < E; ++i) sum[i] += f[i];
            }
        }
    };
    // the places of a token's pairs, in order, by one wave
    auto list = [&](uint32_t key, uint32_t* rows) {
        int n = 0;
        for (int j0 = 0; j0 < m; j0 += 64) {
            const bool its = j0 + lane < m && keys[min(j0 + lane, m - 1)] == key;
            const uint64_t them = __builtin_amdgcn_ballot_w64(its);
            if (its) rows[n + before(them)] = places[j0 + lane];
            n += __builtin_popcountll(them);
        }
        __builtin_amdgcn_wave_barrier();
        return n;
    };
    if (group < groups)
        for (int k = group; k < lights; k += groups) {
            const uint32_t key = light[k] * CLASSES + c;
            const int n = list(key, few_rows[wave]);
            for (int block = first_block; block < blocks; block += across) {
                float sum[E];
                add_rows(few_rows[wave], n, 0, 1, block, sum);
                if (block * 64 + lane < row_pieces) finish(table + (size_t)key * d + (block * 64 + lane) * E, sum, scale, into);
            }
        }
    for (int k = 0; k < heavies; ++k) {
        const uint32_t key = heavy[k] * CLASSES + c;
        const int n = count[heavy[k]];
        if (wave == 0) list(key, many_rows);
        __syncthreads();
        for (int b0 = 0; b0 < blocks; b0 += across) {
            const int block = b0 + first_block;
            float sum[E];
            if (group < groups && block < blocks) add_rows(many_rows, n, group, groups, block, sum);
#pragma unroll
            for (int i = 0; i < E / 4; ++i) sums[wave][i][lane] = f32x4{sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]};
            __syncthreads();
            if (group == 0 && block * 64 + lane < row_pieces) {
                for (int g = 1; g < groups; ++g)
#pragma unroll
                    for (int i = 0; i < E; ++i) sum[i] += sums[g * across + wave][i / 4][lane][i % 4];
                finish(table + (size_t)key * d + (block * 64 + lane) * E, sum, scale, into);
            }
            __syncthreads();
        }
    }
    // the rows of the class that have no token, a wave each
    if (!into)
        for (int q = wave; q < quotients; q += 16)
            if (count[q] == 0) clear_row(table + (size_t)(q * CLASSES + c) * d, row_pieces);
}

// More: a radix sort from the low digit up, two launches a digit.  Workgroup w has the tokens [w each, (w + 1) each); those behind
// clear memory.  The last launch notes which tokens are there.  32768 tokens in four launches 28.7 us, 128 MB cleared beside them.
template <class I, bool FIRST>
struct SortInput {
    const I* ids;
    const u32x2* pairs;
    uint32_t vocab;
    __device__ __forceinline__ u32x2 operator()(int i) const {
        if constexpr (FIRST) return u32x2{min(emb::key_of(ids[i]), vocab), (uint32_t)i};
        else return pairs[i];
    }
};
template <class I, bool FIRST>
__global__ __launch_bounds__(1024) void embedding_count_kernel(SortInput<I, FIRST> in, uint32_t* __restrict__ hist, int n, int each, int workgroups, int at,
                                                               int bits, Zeros zeros, Zeros none, uint32_t none_workgroups) {
    __shared__ uint32_t count[1 << emb::MAX_DIGIT];
    if ((int)blockIdx.x >= workgroups) {
        const uint32_t w = blockIdx.x - workgroups;
        return w < none_workgroups ? none.fill(w) : zeros.fill(w - none_workgroups);
    }
    const int digits = 1 << bits, first = blockIdx.x * each, end = min(n, first + each);
    for (int d = threadIdx.x; d < digits; d += 1024) count[d] = 0;
    __syncthreads();
    for (int i = first + threadIdx.x; i < end; i += 1024) atomicAdd(&count[in(i).x >> at & (digits - 1)], 1u);
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += 1024) hist[blockIdx.x * digits + d] = count[d];
}
template <class I, bool FIRST>
__global__ __launch_bounds__(1024) void embedding_scatter_kernel(SortInput<I, FIRST> in, const uint32_t* __restrict__ hist, u32x2* __restrict__ out,
                                                                 uint8_t* __restrict__ there, int n, uint32_t vocab, int each, int workgroups, int at,
                                                                 int bits, Zeros zeros) {
    constexpr int MOST = 1 << emb::MAX_DIGIT;
    __shared__ uint32_t place[MOST], total[MOST];
    __shared__ uint16_t count[16][MOST];
    if ((int)blockIdx.x >= workgroups) return zeros.fill(blockIdx.x - workgroups);
    const int digits = 1 << bits, first = blockIdx.x * each, end = min(n, first + each);
    for (int d = threadIdx.x; d < 16 * digits; d += 1024) count[d >> bits][d & (digits - 1)] = 0;
    // where this workgroup's tokens of a digit go: behind all smaller digits and the same one of the workgroups in front
    for (int d = threadIdx.x; d < digits; d += 1024) place[d] = total[d] = 0;
    __syncthreads();
    {
        const int d = threadIdx.x & (digits - 1), step = 1024 >> bits;
        uint32_t all = 0, front = 0;
#pragma unroll 8
        for (int w = threadIdx.x >> bits; w < workgroups; w += step) {
            const uint32_t c = hist[w * digits + d];
            all += c;
            front += w < (int)blockIdx.x ? c : 0;
        }
        atomicAdd(&total[d], all);
        atomicAdd(&place[d], front);
    }
    __syncthreads();
    if (threadIdx.x < 64) add_scan(place, total, digits);
    __syncthreads();
    for (int start = first; start < end; start += emb::CHUNK) {
        const int i = start + threadIdx.x;
        const u32x2 pair = i < end ? in(i) : u32x2{0, 0};
        const uint32_t to = take_places(place, count, pair.x >> at & (digits - 1), i < end, bits);
        if (i < end) {
            out[to] = pair;
            if (there && pair.x < vocab) there[pair.x] = 1;
        }
    }
}

// ---- the sums

// The pairs [first - PIECE, first + 2 PIECE) on the lanes of a wave: number o of them on lane o % 64 of register o / 64.
template <int PIECE>
struct Window {
    static constexpr int N = 3 * PIECE, REGS = (N + 63) / 64;
    u32x2 pair[REGS];
    int from;
    __device__ __forceinline__ Window(const u32x2* pairs, int n, int first) : from(first - PIECE) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int r = 0; r < REGS; ++r) {
            const int o = lane + 64 * r, i = from + o;
            pair[r] = o < N && i >= 0 && i < n ? pairs[i] : u32x2{0xffffffffu, 0};
        }
    }
    template <int C>
    __device__ __forceinline__ uint32_t get(int i) const {                  // of a pair, the same one for all lanes
        const int o = i - from;
        uint32_t v = __builtin_amdgcn_readlane(pair[0][C], o & 63);
        if constexpr (REGS > 1) {
            const uint32_t w = __builtin_amdgcn_readlane(pair[REGS - 1][C], o & 63);
            v = o < 64 ? v : w;
        }
        return v;
    }
    __device__ __forceinline__ uint32_t key(int i) const { return get<0>(i); }
    __device__ __forceinline__ uint32_t place(int i) const { return get<1>(i); }
    // how many pairs in [a, b) have this key
    __device__ __forceinline__ int with(uint32_t key, int a, int b) const {
        const int lane = threadIdx.x & 63;
        int n = 0;
#pragma unroll
        for (int r = 0; r < REGS; ++r) {
            const int o = lane + 64 * r;
            n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(o < N && from + o >= a && from + o < b && pair[r].x == key));
        }
        return n;
    }
};

// One wave: 64 lanes of 16 bytes of the rows of PIECE consecutive pairs, and of those of a last run that goes on behind them, if it is no longer
// than PIECE; a run in front that is the wave's before, it leaves out.  Waves behind those of the pieces have a row of the
// table each, of the first `zero_rows`, and clear it where it has no token.
// 32768 tokens of 2048 bf16, 126 MB read and 142 written, 52 us: 5.3 TB/s (with the zeros first 57, in turn with the sums 60).
template <class T, int PIECE, bool CACHED, bool INTO>
__global__ __launch_bounds__(256) void embedding_sum_kernel(const u32x2* __restrict__ pairs, const T* __restrict__ d_out, T* __restrict__ table,
                                                            float* __restrict__ part, int n, uint32_t vocab, int row_pieces, int blocks,
                                                            int tasks, const uint8_t* __restrict__ there, int zero_rows, float scale) {
    using R = emb::Row<T>;
    constexpr int E = R::E;
    const int lane = threadIdx.x & 63, task = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const size_t d = (size_t)row_pieces * E;
    if (task >= tasks) {
        const int row = task - tasks;
        if (row < zero_rows && there[row] == 0) clear_row(table + row * d, row_pieces);
        return;
    }
    const int piece = task / blocks, p = (task % blocks) * 64 + lane;
    const int first = piece * PIECE, end = min(n, first + PIECE);
    const Window<PIECE> w(pairs, n, first);
    const bool has = p < row_pieces;
    const int col = (has ? p : 0) * E;
    int t = first, last = end;                                      // the pairs that are summed here
    uint32_t key = w.key(first);
    bool from_before = first > 0 && w.key(first - 1) == key;        // a long run that began in an earlier piece
    if (from_before) {
        const int more = w.with(key, first, end + PIECE);
        if (w.with(key, first - PIECE, first) + more <= PIECE) {
            from_before = false;
            t = first + more;
            if (t >= end) return;
            key = w.key(t);
        }
    }
    if (key >= vocab) return;                                       // they stand last
    bool goes_on = false;                                           // the last run is long
    if (end < n && w.key(end - 1) == w.key(end)) {
        const int more = w.with(w.key(end), end, end + PIECE);
        if (w.with(w.key(end), first - PIECE, end) + more <= PIECE) last += more; else goes_on = true;
    }
    float sum[E];
#pragma unroll
    for (int i = 0; i < E; ++i) sum[i] = 0.0f;
    // What is there of a row is asked for with the rows that are added to it: 16384 different tokens of 1024 f32 48 us; at the end of each run 58.
    auto old_row = [&](uint32_t key) { return ld_global_16(table + (size_t)min(key, vocab - 1) * d + col); };
    u32x4 old = {0, 0, 0, 0};
    if constexpr (INTO) old = old_row(key);
    auto end_run = [&](bool open) {
        if (key >= vocab || !has) return;
        if (from_before || open) {
            float* to = part + ((size_t)piece * 2 + (from_before ? 0 : 1)) * d + col;
#pragma unroll
            for (int i = 0; i < E; i += 4) *reinterpret_cast<f32x4*>(to + i) = f32x4{sum[i], sum[i + 1], sum[i + 2], sum[i + 3]};
        } else {
            finish<T, INTO>(table + (size_t)key * d + col, sum, scale, old);
        }
    };
    constexpr int AHEAD = INTO ? 8 : 16;      // 32768 tokens of 65536 x 2048 bf16 91 us with 16, 97 with 8; with 8 in turns of two sets 89, but f32 5 % more
    u32x4 row[AHEAD], olds[AHEAD];
    for (; t < last; t += AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            row[u] = ld_stream_16<CACHED>(d_out + (size_t)w.place(min(t + u, last - 1)) * d + col);
            if constexpr (INTO) olds[u] = old_row(w.key(min(t + u, last - 1)));
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (t + u >= last) break;
            const uint32_t k = w.key(t + u);
            if (k != key) {
                end_run(false);
                key = k;
                if constexpr (INTO) old = olds[u];
                from_before = false;
#pragma unroll
                for (int i = 0; i < E; ++i) sum[i] = 0.0f;
            }
            float f[E];
            R::unpack(row[u], f);
#pragma unroll
            for (int i = 0; i < E; ++i) sum[i] += f[i];
        }
    }
    end_run(goes_on);
}

// Four f32 sums to a row of the table.
__device__ __forceinline__ void finish_four(uint16_t* to, f32x4 sum, float scale, bool into) {
    sum *= scale;
    if (into) {
        const u32x2 old = ld_global_8(to);
        sum += f32x4{bf16_lo(old.x), bf16_hi(old.x), bf16_lo(old.y), bf16_hi(old.y)};
    }
    st_global_8(to, u32x2{pack_bf16(sum[0], sum[1]), pack_bf16(sum[2], sum[3])});
}
__device__ __forceinline__ void finish_four(float* to, f32x4 sum, float scale, bool into) {
    sum *= scale;
    if (into) sum += *reinterpret_cast<const f32x4*>(to);
    *reinterpret_cast<f32x4*>(to) = sum;
}

// Long runs: a workgroup looks through 16 pieces, a wave each, for those where one begins, and adds the rows that they left, 256 columns of them:
// the wave itself up to ALONE rows, all waves in turn more of them.  6 us, of which the search is most.
template <class T, int PIECE>
__global__ __launch_bounds__(1024) void embedding_join_kernel(const u32x2* __restrict__ pairs, const float* __restrict__ part, T* __restrict__ table,
                                                              int n, uint32_t vocab, int d_model, int blocks, int pieces, float scale, bool into) {
    constexpr int ALONE = 8;
    __shared__ f32x4 sums[16][64];
    __shared__ uint32_t keys[16];
    __shared__ int lasts[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = ((blockIdx.x % blocks) * 64 + lane) * 4, piece0 = (blockIdx.x / blocks) * 16, mine = piece0 + wave;
    const bool has = col < d_model;
    const size_t d = d_model;
    const float* from = part + (has ? col : 0);
    uint32_t found = 0xffffffffu;
    int last = mine;
    if (mine < pieces - 1) {
        const int first = mine * PIECE, end = first + PIECE;
        const Window<PIECE> w(pairs, n, first);
        // how many of the pieces q, q + step, ... begin with the token, up to 64
        auto begin_with = [&](int q, int step, uint32_t key) {
            const size_t at = ((size_t)q + (size_t)lane * step) * PIECE;
            const uint64_t more = __builtin_amdgcn_ballot_w64(at < (size_t)n && pairs[at < (size_t)n ? at : 0].x == key);
            return ~more ? __builtin_ctzll(~more) : 64;
        };
        const uint32_t key = w.key(end);
        const int here = w.with(key, first, end), more = w.with(key, end, end + PIECE);
        if (key < vocab && here > 0 && here + more > PIECE && !(here == PIECE && first > 0 && w.key(first - 1) == key)) {
            found = key;
            last += begin_with(last + 1, 1, key);
            if (last == mine + 64)                                  // the run's end, 64 times nearer with each look
                for (int left = pieces - 1 - last; left > 0;) {
                    const int step = (left + 63) / 64;
                    last += begin_with(last + step, step, key) * step;
                    left = min(step - 1, pieces - 1 - last);
                }
        }
    }
    const bool alone = found != 0xffffffffu && last - mine < ALONE;
    if (lane == 0) {
        keys[wave] = alone ? 0xffffffffu : found;
        lasts[wave] = last;
    }
    if (alone) {
        f32x4 sum = {0.f, 0.f, 0.f, 0.f}, row[ALONE];
#pragma unroll
        for (int k = 0; k < ALONE; ++k) row[k] = *reinterpret_cast<const f32x4*>(from + ((size_t)min(mine + k, last) * 2 + (k == 0 ? 1 : 0)) * d);
#pragma unroll
        for (int k = 0; k < ALONE; ++k)
            if (mine + k <= last) sum += row[k];
        if (has) finish_four(table + (size_t)found * d + col, sum, scale, into);
    }
    __syncthreads();
    for (int b = 0; b < 16; ++b) {
        const uint32_t key = keys[b];
        if (key == 0xffffffffu) continue;
        const int piece = piece0 + b, end = lasts[b];
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int q = piece + wave; q <= end; q += 16) sum += *reinterpret_cast<const f32x4*>(from + ((size_t)q * 2 + (q == piece ? 1 : 0)) * d);
        sums[wave][lane] = sum;
        __syncthreads();
        if (wave == 0 && has) {
#pragma unroll
            for (int k = 1; k < 16; ++k) sum += sums[k][lane];
            finish_four(table + (size_t)key * d + col, sum, scale, into);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------
namespace {
using namespace emb;
struct Plan {
    bool few, gathered;                   // one launch; pairs by residue classes.  Otherwise a radix sort:
    int digits, bits;                     // passes, bits of each (of the quotients, where they are gathered)
    int each, workgroups;                 // tokens of a workgroup of the sort
    int piece, pieces, blocks;            // pairs of a piece, pieces, 64-lane blocks of a row
    size_t row_pieces;                    // 16-byte pieces of a row
    size_t pairs_bytes, there_bytes, hist_bytes, part_bytes;
    size_t bytes() const { return few ? 0 : (gathered ? 1 : 2) * pairs_bytes + there_bytes + hist_bytes + part_bytes; }
};
int bits_of(size_t v) {
    int bits = 0;
    while (v >> bits) ++bits;
    return bits;
}
Plan plan(size_t n, size_t vocab, size_t d_model, int elem_bytes) {
    Plan p{};
    auto whole = [](size_t b) { return (b + 255) / 256 * 256; };
    p.row_pieces = d_model * elem_bytes / 16;
    p.blocks = (int)((p.row_pieces + 63) / 64);
    const bool classes = vocab <= (size_t)CLASSES * MAX_QUOTIENTS;
    p.few = classes && n * p.blocks <= FEW;
    p.gathered = classes && n <= GATHERED;
    if (p.gathered) {
        p.bits = std::max(1, bits_of((vocab - 1) / CLASSES));
    } else {
        const int bits = bits_of(vocab);  // of a key: the tokens and `vocab`, which stands for those outside of the table
        p.digits = (bits + MAX_DIGIT - 1) / MAX_DIGIT;
        p.bits = (bits + p.digits - 1) / p.digits;
        const size_t chunks = (n + CHUNK - 1) / CHUNK;
        p.each = (int)((chunks + CHUNKS - 1) / CHUNKS * CHUNK);
        p.workgroups = (int)((n + p.each - 1) / p.each);
        p.hist_bytes = whole((size_t)p.workgroups * ((size_t)4 << p.bits));
    }
    // Long pieces where they leave a wave for every SIMD, short ones where they do not, one rule for a whole table and for sums that are added to one.
    // 8192 tokens of 2048 bf16, one wave: a whole table 45.6 us so and 49.8 with pieces of 8 (all one token 51.8 and 62.7), added 29.9 and
    // 27.8 (33.3 and 40.0); 16384 added 41.4 and 44.4 (49.1 and 65.3).  4096, which leave half of the SIMDs without: a whole table 46.0 so and
    // 44.1 with pieces of 32 (49.2 and 44.3), added 22.3 and 28.0 (27.1 and 24.4).
    p.piece = n / 32 * p.blocks >= 1024 ? 32 : 8;
    p.pieces = (int)((n + p.piece - 1) / p.piece);
    p.pairs_bytes = whole(n * 8);
    p.there_bytes = whole(vocab);
    p.part_bytes = p.pieces > 1 ? (size_t)p.pieces * 2 * d_model * 4 : 0;
    return p;
}
}  // namespace

bool embedding_fits(size_t n, int d_model, int elem_bytes) {
    const size_t row_pieces = (size_t)d_model * elem_bytes / 16;
    size_t threads = 1;
    while (threads < row_pieces && threads < 256) threads *= 2;
    return n * threads < ((size_t)1 << 32) - 256;
}

int launch_embedding(const void* ids, int ids64, const void* table, void* out, size_t n, size_t vocab, int d_model, float scale, int bf16,
                     hipStream_t stream) {
    const int pieces = d_model * (bf16 ? 2 : 4) / 16;
    int shift = 0;
    while ((1 << shift) < pieces && shift < 8) ++shift;
    const int rows = 256 >> shift;
    auto go = [&](auto elem, auto index) {
        using T = decltype(elem);
        using I = decltype(index);
        launch_kernel((embedding_kernel<T, I>), dim3((unsigned)((n + rows - 1) / rows)), dim3(256), 0, stream, static_cast<const I*>(ids),
                      static_cast<const T*>(table), static_cast<T*>(out), n, (uint32_t)vocab, pieces, shift, scale);
    };
    if (bf16) { if (ids64) go(uint16_t{}, int64_t{}); else go(uint16_t{}, int32_t{}); }
    else { if (ids64) go(float{}, int64_t{}); else go(float{}, int32_t{}); }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

size_t embedding_bwd_workspace_bytes(size_t n, size_t vocab, int d_model, int bf16) { return plan(n, vocab, d_model, bf16 ? 2 : 4).bytes(); }

bool embedding_bwd_fits(size_t n, size_t vocab, int d_model, int bf16) {
    const Plan p = plan(n, vocab, d_model, bf16 ? 2 : 4);
    // waves of the sums and workgroups of the join
    return (size_t)p.pieces * p.blocks + vocab < ((size_t)1 << 26) &&
           ((size_t)p.pieces + 15) / 16 * ((d_model + 255) / 256) < ((size_t)1 << 22);
}

int launch_embedding_bwd(const void* d_out, const void* ids, int ids64, void* table, size_t n, size_t vocab, int d_model, float scale, int into,
                         int bf16, void* workspace, hipStream_t stream) {
    const Plan p = plan(n, vocab, d_model, bf16 ? 2 : 4);
    const int count = (int)n, row_pieces = d_model * (bf16 ? 2 : 4) / 16;
    auto with_types = [&](auto go) {
        if (bf16) { if (ids64) go(uint16_t{}, int64_t{}); else go(uint16_t{}, int32_t{}); }
        else { if (ids64) go(float{}, int64_t{}); else go(float{}, int32_t{}); }
    };
    if (p.few) {
        with_types([&](auto elem, auto index) {
            using T = decltype(elem);
            using I = decltype(index);
            launch_kernel((embedding_few_kernel<T, I>), dim3(CLASSES), dim3(1024), 0, stream, static_cast<const I*>(ids), static_cast<const T*>(d_out),
                          static_cast<T*>(table), count, (uint32_t)vocab, row_pieces, p.blocks, scale, into != 0);
        });
        return hipGetLastError() == hipSuccess ? 0 : -1;
    }
    char* at = static_cast<char*>(workspace);
    u32x2 *pairs = reinterpret_cast<u32x2*>(at), *other = nullptr;
    at += p.pairs_bytes;
    if (!p.gathered) {
        other = reinterpret_cast<u32x2*>(at);
        at += p.pairs_bytes;
    }
    uint8_t* there = reinterpret_cast<uint8_t*>(at);
    at += p.there_bytes;
    uint32_t* hist = reinterpret_cast<uint32_t*>(at);
    float* part = reinterpret_cast<float*>(at + p.hist_bytes);
    // the last rows of the table, to be cleared beside the sort
    size_t rows = vocab;
    auto last_rows = [&](size_t bytes) {
        const size_t row = p.row_pieces * 16, n = into ? 0 : std::min(rows, bytes / row);
        rows -= n;
        return Zeros{static_cast<char*>(table) + rows * row, n * p.row_pieces};
    };
    with_types([&](auto, auto index) {
        using I = decltype(index);
        const I* from = static_cast<const I*>(ids);
        if (p.gathered) {
            const Zeros zeros = last_rows(BESIDE);
            launch_kernel(embedding_gather_kernel<I>, dim3(CLASSES + zeros.workgroups()), dim3(1024), (size_t)40 << p.bits, stream, from, pairs, there,
                          count, (uint32_t)vocab, p.bits, zeros);
            return;
        }
        for (int k = 0; k < p.digits; ++k) {
            auto pass = [&](auto first) {
                const SortInput<I, first()> in{from, pairs, (uint32_t)vocab};
                const Zeros a = last_rows(BESIDE_PASS), b = last_rows(BESIDE_PASS), none{there, k == 0 && !into ? p.there_bytes / 16 : 0};
                launch_kernel((embedding_count_kernel<I, first()>), dim3(p.workgroups + none.workgroups() + a.workgroups()), dim3(1024), 0, stream, in, hist,
                              count, p.each, p.workgroups, k * p.bits, p.bits, a, none, none.workgroups());
                launch_kernel((embedding_scatter_kernel<I, first()>), dim3(p.workgroups + b.workgroups()), dim3(1024), 0, stream, in, hist, other,
                              k == p.digits - 1 && !into ? there : nullptr, count, (uint32_t)vocab, p.each, p.workgroups, k * p.bits, p.bits, b);
            };
            if (k == 0) pass(std::true_type{}); else pass(std::false_type{});
            std::swap(pairs, other);
        }
    });
    if (hipGetLastError() != hipSuccess) return -1;
    const int tasks = p.pieces * p.blocks, zeros = into ? 0 : (int)rows;
    const bool cached = n * d_model * (bf16 ? 2 : 4) <= kStreamCached;
    auto sums = [&](auto elem, auto piece) {
        using T = decltype(elem);
        auto go = [&](auto in_cache, auto add) {
            launch_kernel((embedding_sum_kernel<T, piece(), in_cache(), add()>), dim3((tasks + zeros + 3) / 4), dim3(256), 0, stream, pairs,
                          static_cast<const T*>(d_out), static_cast<T*>(table), part, count, (uint32_t)vocab, row_pieces, p.blocks, tasks, there, zeros, scale);
        };
        if (cached) { if (into) go(std::true_type{}, std::true_type{}); else go(std::true_type{}, std::false_type{}); }
        else { if (into) go(std::false_type{}, std::true_type{}); else go(std::false_type{}, std::false_type{}); }
        if (p.pieces > 1)
            launch_kernel((embedding_join_kernel<T, piece()>), dim3((p.pieces + 15) / 16 * ((d_model + 255) / 256)), dim3(1024), 0, stream, pairs, part,
                          static_cast<T*>(table), count, (uint32_t)vocab, d_model, (d_model + 255) / 256, p.pieces, scale, into != 0);
    };
    auto of_type = [&](auto elem) {
        if (p.piece == 8) sums(elem, std::integral_constant<int, 8>{}); else sums(elem, std::integral_constant<int, 32>{});
    };
    if (bf16) of_type(uint16_t{}); else of_type(float{});
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tyr
