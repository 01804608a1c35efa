// Embedding: rows of a table by token, and the gradient of the table (gfx950).
//
//   out[i] = scale table[ids[i]]                          a token outside of the table (padding) gives a row of zeros
//   G[v]   = scale sum over i with ids[i] = v of d_out[i]  (or that added to a gradient that is there); such a token adds nothing
//
// The gradient is summed by sorted tokens: no atomic additions of floating point, the same bits every time.  The pairs (token, place) are
// sorted by token, stable; a wave adds the rows of PIECE consecutive pairs, 16 bytes of a row a lane, in f32; a token whose pairs lie in one
// piece is written there, others leave an f32 row for each piece that they reach into, and a last launch adds those.
//
// Bound by HBM: the lookup reads and writes its rows, the gradient reads d_out and writes the table once (zeros for the tokens that are not
// there), or reads and writes the tokens' rows only.
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

constexpr int RANKED = 8192;              // so many tokens at most are sorted by counting
constexpr int CHUNK = 1024, CHUNKS = 128; // radix sort: tokens of a turn, workgroups at most
constexpr int MAX_DIGIT = 9;
constexpr int ZERO_ROWS = 16;             // rows of the table that one wave fills with zeros
constexpr int JOIN_WAVES = 8;
}  // namespace emb

// 2^shift threads a row, 256 >> shift rows a workgroup.
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

// A few tokens: a token's place is how many stand in front of it.  A workgroup has 64 tokens, one a lane; its 16 waves count over groups of 64
// keys in turn, which they read as scalars: a comparison and an addition with carry for 64 pairs of tokens.
template <class I>
__global__ __launch_bounds__(1024) void embedding_rank_kernel(const I* __restrict__ ids, u32x2* __restrict__ pairs, int n) {
    __shared__ int before[16][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), block = blockIdx.x;
    const int i = block * 64 + lane;
    const uint32_t key = emb::key_of(ids[min(i, n - 1)]);
    int count = 0;
    for (int q = wave; q * 64 < n; q += 16) {
        const I* k = ids + q * 64;
        const int m = min(64, n - q * 64);
        if (q == block) {
            for (int j = 0; j < m; ++j) {
                const uint32_t other = emb::key_of(k[j]);
                count += other < key || (other == key && j < lane);
            }
        } else if (q < block) {                                     // equal tokens in front count, those behind do not
#pragma unroll 16
            for (int j = 0; j < 64; ++j) count += emb::key_of(k[j]) <= key;
        } else if (m == 64) {
#pragma unroll 16
            for (int j = 0; j < 64; ++j) count += emb::key_of(k[j]) < key;
        } else {
            for (int j = 0; j < m; ++j) count += emb::key_of(k[j]) < key;      // the last group
        }
    }
    before[wave][lane] = count;
    __syncthreads();
    if (threadIdx.x < 64 && i < n) {
        int rank = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) rank += before[w][lane];
        pairs[rank] = u32x2{key, (uint32_t)i};
    }
}

// Many tokens: a radix sort from the low digit up, two launches a digit.  Workgroup w has the tokens [w each, (w + 1) each).
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
__global__ __launch_bounds__(1024) void embedding_count_kernel(SortInput<I, FIRST> in, uint32_t* __restrict__ hist, int n, int each, int at, int bits) {
    __shared__ uint32_t count[1 << emb::MAX_DIGIT];
    const int digits = 1 << bits, first = blockIdx.x * each, end = min(n, first + each);
    for (int d = threadIdx.x; d < digits; d += 1024) count[d] = 0;
    __syncthreads();
    for (int i = first + threadIdx.x; i < end; i += 1024) atomicAdd(&count[in(i).x >> at & (digits - 1)], 1u);
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += 1024) hist[blockIdx.x * digits + d] = count[d];
}
template <class I, bool FIRST>
__global__ __launch_bounds__(1024) void embedding_scatter_kernel(SortInput<I, FIRST> in, const uint32_t* __restrict__ hist, u32x2* __restrict__ out,
                                                                 int n, int each, int at, int bits) {
    constexpr int MOST = 1 << emb::MAX_DIGIT;
    __shared__ uint32_t place[MOST], total[MOST], count[16][MOST];
    const int digits = 1 << bits, first = blockIdx.x * each, end = min(n, first + each), workgroups = gridDim.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
    if (wave == 0) {
        uint32_t sum = 0;
        const int each_lane = max(1, digits / 64), d0 = lane * each_lane;
        if (d0 < digits)
            for (int k = 0; k < each_lane; ++k) sum += total[d0 + k];
        uint32_t front = sum;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t other = __shfl_up(front, o, 64);
            if (lane >= o) front += other;
        }
        front -= sum;
        if (d0 < digits)
            for (int k = 0; k < each_lane; ++k) {
                place[d0 + k] += front;
                front += total[d0 + k];
            }
    }
    for (int start = first; start < end; start += emb::CHUNK) {
        for (int d = threadIdx.x; d < 16 * digits; d += 1024) count[d >> bits][d & (digits - 1)] = 0;
        __syncthreads();
        const int i = start + threadIdx.x;
        const bool real = i < end;
        const u32x2 pair = real ? in(i) : u32x2{0, 0};
        const int digit = pair.x >> at & (digits - 1);
        // the lanes that have the same digit
        uint64_t same = __builtin_amdgcn_ballot_w64(real);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __builtin_amdgcn_ballot_w64(digit >> b & 1);
            same &= digit >> b & 1 ? set : ~set;
        }
        const int rank = __builtin_popcountll(same & (((uint64_t)1 << lane) - 1));
        if (real && rank == 0) count[wave][digit] = __builtin_popcountll(same);
        __syncthreads();
        for (int d = threadIdx.x; d < digits; d += 1024) {
            uint32_t to = place[d];
#pragma unroll
            for (int w = 0; w < 16; ++w) {
                const uint32_t c = count[w][d];
                count[w][d] = to;
                to += c;
            }
            place[d] = to;
        }
        __syncthreads();
        if (real) out[count[wave][digit] + rank] = pair;
        __syncthreads();
    }
}

// ---- the sums

// first of the sorted pairs whose key is not below `key`
__device__ __forceinline__ int first_of(const u32x2* pairs, int n, uint32_t key) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (pairs[mid].x < key) lo = mid + 1; else hi = mid;
    }
    return lo;
}
// A sum as it goes to the table's row.
template <class T>
__device__ __forceinline__ void finish(T* to, float (&sum)[emb::Row<T>::E], float scale, bool into) {
    using R = emb::Row<T>;
#pragma unroll
    for (int i = 0; i < R::E; ++i) sum[i] *= scale;
    if (into) {
        float old[R::E];
        R::unpack(ld_global_16(to), old);
#pragma unroll
        for (int i = 0; i < R::E; ++i) sum[i] += old[i];
    }
    st_global_16_nt(to, R::pack(sum));
}

// One wave: 64 lanes of 16 bytes of PIECE consecutive pairs' rows.  Waves behind those of the pieces fill ZERO_ROWS rows of the table each with
// zeros, where no pair has them.
template <class T, int PIECE>
__global__ __launch_bounds__(256) void embedding_sum_kernel(const u32x2* __restrict__ pairs, const T* __restrict__ d_out, T* __restrict__ table,
                                                            float* __restrict__ part, int n, uint32_t vocab, int row_pieces, int blocks,
                                                            int piece_tasks, float scale, bool into) {
    using R = emb::Row<T>;
    constexpr int E = R::E;
    const int lane = threadIdx.x & 63, task = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const size_t d = (size_t)row_pieces * E;
    if (task >= piece_tasks) {
        const uint32_t v0 = (uint32_t)(task - piece_tasks) * emb::ZERO_ROWS;
        if (into || v0 >= vocab) return;
        bool there = true;
        if (lane < emb::ZERO_ROWS && v0 + lane < vocab) {
            const int at = first_of(pairs, n, v0 + lane);
            there = at < n && pairs[at].x == v0 + lane;
        }
        uint64_t absent = __builtin_amdgcn_ballot_w64(!there);
        while (absent) {
            const int r = __builtin_ctzll(absent);
            absent &= absent - 1;
            T* to = table + (size_t)(v0 + r) * d;
            for (int p = lane; p < row_pieces; p += 64) st_global_16_nt(to + p * E, u32x4{0, 0, 0, 0});
        }
        return;
    }
    const int piece = task / blocks, p = (task % blocks) * 64 + lane;
    const int first = piece * PIECE, count = min(PIECE, n - first);
    const bool has = p < row_pieces;
    const int col = (has ? p : 0) * E;
    const u32x2 mine = pairs[first + min(lane, count - 1)];
    const uint32_t before = first > 0 ? pairs[first - 1].x : 0xffffffffu, behind = first + count < n ? pairs[first + count].x : 0xffffffffu;
    uint32_t key = __builtin_amdgcn_readlane(mine.x, 0);
    if (key >= vocab) return;                                       // they stand last
    bool from_before = first > 0 && before == key;                  // the run that is being summed began in an earlier piece
    float sum[E];
#pragma unroll
    for (int i = 0; i < E; ++i) sum[i] = 0.0f;
    auto end_run = [&](bool goes_on) {
        if (key >= vocab || !has) return;
        if (from_before || goes_on) {
            float* to = part + ((size_t)piece * 2 + (from_before ? 0 : 1)) * d + col;
#pragma unroll
            for (int i = 0; i < E; i += 4) *reinterpret_cast<f32x4*>(to + i) = f32x4{sum[i], sum[i + 1], sum[i + 2], sum[i + 3]};
        } else {
            finish(table + (size_t)key * d + col, sum, scale, into);
        }
    };
    constexpr int AHEAD = 8;
    u32x4 row[AHEAD];
    for (int t = 0; t < count; t += AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const uint32_t at = __builtin_amdgcn_readlane(mine.y, min(t + u, count - 1));
            row[u] = ld_global_16_nt(d_out + (size_t)at * d + col);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (t + u >= count) break;
            const uint32_t k = __builtin_amdgcn_readlane(mine.x, t + u);
            if (k != key) {
                end_run(false);
                key = k;
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
    end_run(behind == key);
}

// Runs of one token over several pieces: workgroup (piece, 64 lanes of 16 bytes) where one begins adds its rows, by waves in turn.
template <class T, int PIECE>
__global__ __launch_bounds__(64 * emb::JOIN_WAVES) void embedding_join_kernel(const u32x2* __restrict__ pairs, const float* __restrict__ part,
                                                                              T* __restrict__ table, int n, uint32_t vocab, int row_pieces,
                                                                              int blocks, float scale, bool into) {
    using R = emb::Row<T>;
    constexpr int E = R::E, WAVES = emb::JOIN_WAVES;
    __shared__ f32x4 sums[WAVES][E / 4][64];
    const int piece = blockIdx.x / blocks, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, p = (blockIdx.x % blocks) * 64 + lane;
    const int next = (piece + 1) * PIECE;                           // a pair: there is another piece
    const uint32_t key = pairs[next].x;
    if (key >= vocab || pairs[next - 1].x != key || (piece > 0 && pairs[next - PIECE - 1].x == key && pairs[next - PIECE].x == key)) return;
    const size_t d = (size_t)row_pieces * E;
    const bool has = p < row_pieces;
    const int col = (has ? p : 0) * E;
    // pieces that begin with the token: behind this one, up to `last`
    int last = piece + 1;
    for (int q = piece + 2;; q += 64) {
        const size_t at = (size_t)(q + lane) * PIECE;
        const uint64_t more = __builtin_amdgcn_ballot_w64(at < (size_t)n && pairs[at < (size_t)n ? at : 0].x == key);
        const int m = ~more ? __builtin_ctzll(~more) : 64;
        last += m;
        if (m < 64) break;
    }
    f32x4 sum[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int q = piece + wave; q <= last; q += WAVES) {
        const float* from = part + ((size_t)q * 2 + (q == piece ? 1 : 0)) * d + col;
#pragma unroll
        for (int i = 0; i < E / 4; ++i) sum[i] += *reinterpret_cast<const f32x4*>(from + 4 * i);
    }
#pragma unroll
    for (int i = 0; i < E / 4; ++i) sums[wave][i][lane] = sum[i];
    __syncthreads();
    if (wave != 0 || !has) return;
    float total[E];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
#pragma unroll
        for (int w = 1; w < WAVES; ++w) sum[i] += sums[w][i][lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) total[4 * i + j] = sum[i][j];
    }
    finish(table + (size_t)key * d + col, total, scale, into);
}

// ------------------------------------------------------------------------------------------
namespace {
using namespace emb;
struct Plan {
    int digits, bits;                     // radix sort: passes, bits of each; 0 = by counting
    int each, workgroups;                 // tokens of a workgroup of the sort
    int piece, pieces, blocks;            // pairs of a piece, pieces, 64-lane blocks of a row
    size_t pairs_bytes, hist_bytes, part_bytes;
    size_t bytes() const { return (digits ? 2 : 1) * pairs_bytes + hist_bytes + part_bytes; }
};
Plan plan(size_t n, size_t vocab, size_t d_model, int elem_bytes) {
    Plan p{};
    auto whole = [](size_t b) { return (b + 255) / 256 * 256; };
    if (n > RANKED) {
        int bits = 0;                     // of a key: the tokens and `vocab`, which stands for those outside of the table
        while (bits < 32 && vocab >> bits) ++bits;
        p.digits = (bits + MAX_DIGIT - 1) / MAX_DIGIT;
        p.bits = (bits + p.digits - 1) / p.digits;
        const size_t chunks = (n + CHUNK - 1) / CHUNK;
        p.each = (int)((chunks + CHUNKS - 1) / CHUNKS * CHUNK);
        p.workgroups = (int)((n + p.each - 1) / p.each);
        p.hist_bytes = whole((size_t)p.workgroups * ((size_t)4 << p.bits));
    }
    p.piece = n > RANKED ? 32 : 8;
    p.pieces = (int)((n + p.piece - 1) / p.piece);
    const size_t row_pieces = d_model * elem_bytes / 16;
    p.blocks = (int)((row_pieces + 63) / 64);
    p.pairs_bytes = whole(n * 8);
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
    const size_t tasks = (size_t)p.pieces * p.blocks, zeros = (vocab + ZERO_ROWS - 1) / ZERO_ROWS;
    return tasks + zeros < ((size_t)1 << 26) && tasks * JOIN_WAVES < ((size_t)1 << 26);
}

int launch_embedding_bwd(const void* d_out, const void* ids, int ids64, void* table, size_t n, size_t vocab, int d_model, float scale, int into,
                         int bf16, void* workspace, hipStream_t stream) {
    const Plan p = plan(n, vocab, d_model, bf16 ? 2 : 4);
    char* at = static_cast<char*>(workspace);
    u32x2 *pairs = reinterpret_cast<u32x2*>(at), *other = nullptr;
    at += p.pairs_bytes;
    if (p.digits) {
        other = reinterpret_cast<u32x2*>(at);
        at += p.pairs_bytes;
    }
    uint32_t* hist = reinterpret_cast<uint32_t*>(at);
    float* part = reinterpret_cast<float*>(at + p.hist_bytes);
    const int count = (int)n;
    auto sort = [&](auto index) {
        using I = decltype(index);
        const I* from = static_cast<const I*>(ids);
        if (!p.digits) {
            launch_kernel(embedding_rank_kernel<I>, dim3((count + 63) / 64), dim3(1024), 0, stream, from, pairs, count);
            return;
        }
        for (int k = 0; k < p.digits; ++k) {
            auto pass = [&](auto first) {
                const SortInput<I, first()> in{from, pairs, (uint32_t)vocab};
                launch_kernel((embedding_count_kernel<I, first()>), dim3(p.workgroups), dim3(1024), 0, stream, in, hist, count, p.each, k * p.bits, p.bits);
                launch_kernel((embedding_scatter_kernel<I, first()>), dim3(p.workgroups), dim3(1024), 0, stream, in, hist, other, count, p.each,
                              k * p.bits, p.bits);
            };
            if (k == 0) pass(std::true_type{}); else pass(std::false_type{});
            std::swap(pairs, other);
        }
    };
    if (ids64) sort(int64_t{}); else sort(int32_t{});
    if (hipGetLastError() != hipSuccess) return -1;
    const int tasks = p.pieces * p.blocks, zeros = into ? 0 : (int)((vocab + ZERO_ROWS - 1) / ZERO_ROWS);
    const int row_pieces = d_model * (bf16 ? 2 : 4) / 16;
    auto sums = [&](auto elem, auto piece) {
        using T = decltype(elem);
        launch_kernel((embedding_sum_kernel<T, piece()>), dim3((tasks + zeros + 3) / 4), dim3(256), 0, stream, pairs, static_cast<const T*>(d_out),
                      static_cast<T*>(table), part, count, (uint32_t)vocab, row_pieces, p.blocks, tasks, scale, into != 0);
        if (p.pieces > 1)
            launch_kernel((embedding_join_kernel<T, piece()>), dim3(tasks - p.blocks), dim3(64 * JOIN_WAVES), 0, stream, pairs, part,
                          static_cast<T*>(table), count, (uint32_t)vocab, row_pieces, p.blocks, scale, into != 0);
    };
    auto of_type = [&](auto elem) {
        if (p.piece == 8) sums(elem, std::integral_constant<int, 8>{}); else sums(elem, std::integral_constant<int, 32>{});
    };
    if (bf16) of_type(uint16_t{}); else of_type(float{});
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tyr
