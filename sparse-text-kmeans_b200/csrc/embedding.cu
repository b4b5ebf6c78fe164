// Rows of an embedding table and their gradient.
//
//   out[i, :] = scale * table[id_i, :]            dtable[v, :] = scale * sum over i with id_i = v of grad[i, :]
//
// An id outside [0, rows) - the library's "no node" among them - is no row: zeros, and no gradient.  Sums are held in fp32
// and rounded to the output's type once.  The order of every sum is fixed by the ids, the length of a row and the type of
// `grad`, so that a gradient repeats bit for bit, wherever its matrices lie: nothing is added by atomics.
#include "operators_common.cuh"

namespace cpb {
namespace {

using namespace op;

// ---- lookup -----------------------------------------------------------------------------------------------------------
// A warp takes kLookupVecs * 32 accesses of a row, all of them in flight before the first is stored.  Memory bounds it: 65,536
// tokens of 1,024 bf16 values, as frequent as words are, 29 us, 134 MB written (41 us if every row came from memory); one token
// 2.2 us, an empty kernel's time.
constexpr int kLookupVecs = 4;
constexpr int kLookupThreads = 256;

struct LookupArgs {
    const void* table;
    void* out;
    Ids ids;
    uint64_t n, table_stride, out_stride;  // strides in elements
    uint32_t dim, parts;                   // parts: warps that share a row
    float scale;
};

template <class T, int E>
__global__ void __launch_bounds__(kLookupThreads) lookup_kernel(LookupArgs a) {
    const int lane = threadIdx.x & 31;
    const uint64_t item = (uint64_t(blockIdx.x) * kLookupThreads + threadIdx.x) >> 5;
    const uint64_t row = item / a.parts;
    if (row >= a.n) return;
    const uint32_t id = a.ids.at(row);
    const uint32_t vecs = a.dim / E, v0 = uint32_t(item % a.parts) * (kLookupVecs * 32) + lane;
    const T* src = static_cast<const T*>(a.table) + uint64_t(id == kFull ? 0 : id) * a.table_stride;
    T* dst = static_cast<T*>(a.out) + row * a.out_stride;
    Pack<T, E> x[kLookupVecs];
#pragma unroll
    for (int j = 0; j < kLookupVecs; ++j) {
#pragma unroll
        for (int w = 0; w < Pack<T, E>::kWords; ++w) x[j].raw[w] = typename Pack<T, E>::Raw{};
        if (v0 + j * 32 < vecs && id != kFull) x[j].load(src + size_t(v0 + j * 32) * E);
    }
#pragma unroll
    for (int j = 0; j < kLookupVecs; ++j) {
        if (v0 + j * 32 >= vecs) break;
        // (a row that is none stays the zeros that it was, whatever the scale)
        if (id != kFull) {
#pragma unroll
            for (int e = 0; e < E; ++e) x[j].set(e, x[j].get(e) * a.scale);
        }
        x[j].store(dst + size_t(v0 + j * 32) * E);
    }
    // what is left of a row whose length is no multiple of E
    const uint32_t tail = vecs * E + lane;
    if (item % a.parts == 0 && tail < a.dim) dst[tail] = from_float<T>(id == kFull ? 0.0f : to_float(src[tail]) * a.scale);
}

template <class T, int E>
int launch_lookup(LookupArgs& a, cudaStream_t st) {
    const uint32_t vecs = a.dim / E;
    a.parts = vecs <= kLookupVecs * 32 ? 1 : (vecs + kLookupVecs * 32 - 1) / (kLookupVecs * 32);
    constexpr uint64_t kWarps = kLookupThreads / 32;
    const uint64_t blocks = (a.n * a.parts + kWarps - 1) / kWarps;
    CPB_OP_CHECK(blocks < (1ull << 31), "embedding_lookup: too many rows for one call");
    lookup_kernel<T, E><<<unsigned(blocks), kLookupThreads, 0, st>>>(a);
    CPB_CUDA(cudaGetLastError());
    return 0;
}

template <class T>
int pick_lookup(LookupArgs& a, cudaStream_t st) {
    Alignment al;
    al.add(a.table).add(a.out).add(a.table_stride * sizeof(T)).add(a.out_stride * sizeof(T));
    constexpr int kWide = 16 / sizeof(T);
    if (al.holds(16)) return launch_lookup<T, kWide>(a, st);
    if (al.holds(8)) return launch_lookup<T, kWide / 2>(a, st);
    if (al.holds(4)) return launch_lookup<T, kWide / 4>(a, st);
    return launch_lookup<T, 1>(a, st);
}

// ---- gradient ---------------------------------------------------------------------------------------------------------
// Accesses: E elements of a row of `grad` and as many of `out`; a thread takes the vectors v of a row's dim / E, and the
// last elements, when E does not divide dim, one by one (launches with E > 1 ask that it does).
struct GradArgs {
    Ids ids;
    const void* grad;
    void* out;
    uint64_t grad_stride, out_stride;
    uint32_t n, rows, dim;
    int accumulate;
    float scale;
    uint32_t most_groups;   // form without the sort: groups of threads that a row's places are dealt to, at most
    // sorted form
    uint32_t* pos;          // [n] places in order of (id, place)
    uint32_t* key;          // [n] their ids; `rows` for those that are none
    uint2* range;           // [rows] first and past-the-last place of a row's run, where it has one
    float* partial;         // [n / kRun + 1][2][dim] sums of the pieces of runs longer than kRun
    uint32_t* arrived;      // [kJoinLevels][n / kRun + 1][2][parts] how many of a group are there, under its first piece
    uint32_t parts;         // warps that share a row
    uint32_t piece_blocks;  // the first blocks of the sums' launch, which take pieces of long runs
};

template <class TO, int E>
__device__ __forceinline__ void write_sum(const GradArgs& a, TO* dst, const float (&sum)[E]) {
    Pack<TO, E> o;
    if (a.accumulate) {
        o.load(dst);
#pragma unroll
        for (int e = 0; e < E; ++e) o.set(e, o.get(e) + sum[e] * a.scale);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) o.set(e, sum[e] * a.scale);
    }
    o.store(dst);
}

// A row of zeros, by `threads` threads.  E elements are 16 bytes or 32, or fewer where the output is not aligned to 16.
template <class TO, int E>
__device__ __forceinline__ void clear_row(const GradArgs& a, uint64_t row, uint32_t thread, uint32_t threads) {
    constexpr int kE = E * int(sizeof(TO)) > 16 ? 16 / int(sizeof(TO)) : E;
    TO* dst = static_cast<TO*>(a.out) + row * a.out_stride;
    Pack<TO, kE> zero;
    zero.raw[0] = typename Pack<TO, kE>::Raw{};
#pragma unroll 4
    for (uint32_t v = thread; v < a.dim / kE; v += threads) zero.store(dst + size_t(v) * kE);
}

// Few tokens, no sort: a block per place.  The block of a row's first place gathers the places behind it that hold the same
// id and sums them; the others end.  Other blocks of the same launch clear the rows that no place names, each reading all
// ids for the rows of its own.  Writes bound it: 512 tokens, 32,768 rows of 1,024 fp32 values, 24 us (the memory needs 21).
constexpr int kSmallLog = 8, kSmallThreads = 1 << kSmallLog;
// Up to kSmallMost places.  (Without the sort, and with it: 2,048 tokens, 4,096 rows of 256 bf16 values 11.5 us and 27;
// 32,768 rows of 1,024 values 25 and 34; 4,096 tokens 22 and 27, 56 and 36.)
constexpr uint32_t kSmallMost = 2048;
constexpr uint32_t kClearRows = 32;    // rows a clearing block owns

template <class TI, class TO, int E>
__global__ void __launch_bounds__(kSmallThreads) grad_small_kernel(GradArgs a) {
    __shared__ uint32_t list[kSmallMost];
    __shared__ uint32_t warp_count[kSmallThreads / 32 + 1];
    __shared__ float sums[kSmallThreads * E];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t vecs = a.dim / E;
    if (blockIdx.x >= a.n) {
        uint32_t* named = list;  // bits of the block's rows
        const uint64_t row0 = uint64_t(blockIdx.x - a.n) * kClearRows;
        if (tid < kClearRows / 32) named[tid] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < a.n; i += kSmallThreads) {
            const uint64_t id = a.ids.at(i);
            if (id >= row0 && id < row0 + kClearRows) atomicOr(&named[uint32_t(id - row0) >> 5], 1u << (uint32_t(id - row0) & 31));
        }
        __syncthreads();
        for (uint32_t r = warp; r < kClearRows && row0 + r < a.rows; r += kSmallThreads / 32)
            if (!(named[r >> 5] >> (r & 31) & 1)) clear_row<TO, E>(a, row0 + r, lane, 32);
        return;
    }
    const uint32_t me = blockIdx.x, id = a.ids.at(me);
    if (id == kFull) return;
    uint32_t before = 0;
    for (uint32_t i = tid; i < me; i += kSmallThreads) before |= a.ids.at(i) == id;
    if (__syncthreads_or(before)) return;
    uint32_t count = 0;
    for (uint32_t i0 = me; i0 < a.n; i0 += kSmallThreads) {
        const uint32_t i = i0 + tid;
        const bool same = i < a.n && a.ids.at(i) == id;
        const uint32_t votes = __ballot_sync(kFull, same);
        if (lane == 0) warp_count[warp] = __popc(votes);
        __syncthreads();
        uint32_t at = count + __popc(votes & ((1u << lane) - 1));
        for (uint32_t w = 0; w < kSmallThreads / 32; ++w) {
            at += w < warp ? warp_count[w] : 0;
            count += warp_count[w];
        }
        if (same) list[at] = i;
        __syncthreads();
    }
    // the places of the list are dealt to groups of threads, a power of two of them along the row
    const uint32_t groups = min(a.most_groups, count), across_log = kSmallLog - (32 - __clz(groups - 1)), across = 1u << across_log;
    const uint32_t group = tid >> across_log;
    const TI* grad = static_cast<const TI*>(a.grad);
    for (uint32_t v0 = 0; v0 < vecs; v0 += across) {
        const uint32_t v = v0 + (tid & (across - 1));
        float sum[E];
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] = 0.0f;
        if (v < vecs && group < groups) {
#pragma unroll 4
            for (uint32_t j = group; j < count; j += groups) {
                Pack<TI, E> x;
                x.load(grad + list[j] * a.grad_stride + size_t(v) * E);
#pragma unroll
                for (int e = 0; e < E; ++e) sum[e] += x.get(e);
            }
        }
        if (groups > 1) {
#pragma unroll
            for (int e = 0; e < E; ++e) sums[tid * E + e] = sum[e];
            __syncthreads();
            if (group == 0)
                for (uint32_t g = 1; g < groups; ++g)
#pragma unroll
                    for (int e = 0; e < E; ++e) sum[e] += sums[(g * across + tid) * E + e];
            __syncthreads();
        }
        if (group == 0 && v < vecs) write_sum<TO, E>(a, static_cast<TO*>(a.out) + id * a.out_stride + size_t(v) * E, sum);
    }
}

// Sorting (id, place): a stable radix sort by digits of up to 9 bits, lowest first.  A pass places the pairs of tiles of
// kSortTile: base of the digit, plus those in tiles before, plus those in warps before, plus the rank among the warp's own; the
// next pass's counts are added up (whole numbers: in any order the same) by those that place.  (All of it in the shared memory
// of one cluster of eight blocks took 94 us for 131,072 ids of 18 bits: ranks and scattered writes want all SMs.  This way 27,
// a chain of launches whose blocks wait for memory a few times each.)
// The first count also marks the rows that are named.  In the launches behind it the blocks that the sort leaves idle clear
// those that are not.
constexpr int kSortThreads = 256, kSortWarps = kSortThreads / 32, kSortRounds = 4;
constexpr uint32_t kSortTile = kSortThreads * kSortRounds;
constexpr int kDigitBits = 9;
constexpr uint32_t kDigits = 1u << kDigitBits;
constexpr uint32_t kGroup = 16;        // tiles whose counts are also held together
constexpr uint32_t kAtOnce = 16;       // of these, read at a time
// Up to kFoldTiles a tile sums the counts of those before it by itself; beyond, a launch per pass does it for all.  (Rows of
// 8 bf16 values, 100,003 of them: 65,536 tokens 50 us and 52, 1,048,576 tokens 304 and 300, 4,194,304 tokens 1,312 and 1,170.)
constexpr uint32_t kFoldTiles = 1024;
constexpr uint32_t kRun = 32;              // a run of equal ids longer than this is summed in pieces, by many warps
constexpr uint32_t kJoin = 16;             // pieces that are joined at a time, and so on
constexpr int kJoinLevels = 3;             // (the last one takes all that are left: 131,072 places are 4,096 pieces or fewer)

// The lanes whose digit is this lane's, among those of `there`, by a vote for each of its bits.
__device__ __forceinline__ uint32_t same_digit(uint32_t digit, bool there) {
    uint32_t same = __ballot_sync(kFull, there);
#pragma unroll
    for (int b = 0; b < kDigitBits; ++b) {
        const uint32_t votes = __ballot_sync(kFull, digit >> b & 1);
        same &= digit >> b & 1 ? votes : ~votes;
    }
    return same;
}

struct SortArgs {
    uint32_t tiles;
    int shift, first, last;
    const uint32_t *key_in, *pos_in;
    uint32_t *key_out, *pos_out;
    uint32_t *counts, *groups;            // [tiles][kDigits] of this pass, [tiles / kGroup + 1][kDigits]
    uint32_t *next_counts, *next_groups;  // of the next one
    uint32_t* totals;  // [kDigits], when the counts have been summed over the tiles by a launch of their own
    uint32_t* named;   // [rows] 1: some place names it
    uint64_t clear0, clear1;  // rows that the blocks behind the tiles clear where they are not named
};

constexpr uint32_t kClearWarpRows = 8;
// Rows that no place names, a few a warp, by the blocks of a launch from `block0` on
template <class TO, int E>
__device__ __forceinline__ void clear_unnamed(const GradArgs& a, const SortArgs& s, uint32_t block0) {
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t row0 = s.clear0 + ((uint64_t(blockIdx.x - block0) * kSortThreads + threadIdx.x) >> 5) * kClearWarpRows;
    if (row0 >= s.clear1) return;
    const uint32_t left = uint32_t(min(uint64_t(kClearWarpRows), s.clear1 - row0));
    for (uint32_t idle = __ballot_sync(kFull, lane < left && !s.named[row0 + lane]); idle; idle &= idle - 1)
        clear_row<TO, E>(a, row0 + __ffs(idle) - 1, lane, 32);
}

__device__ __forceinline__ uint32_t sort_key(const GradArgs& a, const SortArgs& s, uint32_t i) {
    if (!s.first) return s.key_in[i];
    const uint32_t id = a.ids.at(i);
    return id == kFull ? a.rows : id;
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(GradArgs a, SortArgs s) {
    __shared__ uint32_t count[kDigits], keys[kSortTile];
    __shared__ uint16_t last[kSortTile];
    for (uint32_t d = threadIdx.x; d < kDigits; d += kSortThreads) count[d] = 0;
    const uint32_t i0 = blockIdx.x * kSortTile;
    auto slot = [](uint32_t key) { return key * 0x9e3779b1u >> 22; };
    static_assert(kSortTile == 1024, "a slot has 10 bits");
    uint32_t key[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const uint32_t at = r * kSortThreads + threadIdx.x;
        keys[at] = key[r] = i0 + at < a.n ? sort_key(a, s, i0 + at) : kFull;
        last[slot(key[r])] = uint16_t(at);
    }
    __syncthreads();
    // a row is marked by the place that has won its slot, and by those that lost it to another row's: marks that many threads
    // write hold memory up (131,072 places, 64 a row: marked by all, in bytes, 20 us; this way, in words, 9)
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r)
        if (key[r] != kFull) {
            const uint32_t won = last[slot(key[r])];
            atomicAdd(&count[key[r] & (kDigits - 1)], 1u);
            if (key[r] != a.rows && (won == r * kSortThreads + threadIdx.x || keys[won] != key[r])) s.named[key[r]] = 1;
        }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < kDigits; d += kSortThreads) {
        s.counts[size_t(blockIdx.x) * kDigits + d] = count[d];
        if (count[d]) atomicAdd(&s.groups[size_t(blockIdx.x / kGroup) * kDigits + d], count[d]);
    }
}

// counts[t][d] -> those in tiles before t; totals[d].  32 digits a block, the tiles in 32 runs.
__global__ void __launch_bounds__(1024) sort_scan_kernel(uint32_t* counts, uint32_t* totals, uint32_t tiles) {
    __shared__ uint32_t run[32][33];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = blockIdx.x * 32 + lane;
    const uint32_t per = (tiles + 31) / 32, t0 = min(tiles, warp * per), t1 = min(tiles, t0 + per);
    uint32_t sum = 0;
#pragma unroll 8
    for (uint32_t t = t0; t < t1; ++t) sum += counts[size_t(t) * kDigits + d];
    run[warp][lane] = sum;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (uint32_t w = 0; w < 32; ++w) {
        before += w < warp ? run[w][lane] : 0;
        all += run[w][lane];
    }
#pragma unroll 8
    for (uint32_t t = t0; t < t1; ++t) {
        const uint32_t c = counts[size_t(t) * kDigits + d];
        counts[size_t(t) * kDigits + d] = before;
        before += c;
    }
    if (warp == 0) totals[d] = all;
}

template <class TO, int E>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(GradArgs a, SortArgs s) {
    __shared__ uint32_t count[kSortWarps][kDigits];
    __shared__ uint32_t warp_sum[kSortWarps];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (blockIdx.x >= s.tiles) return clear_unnamed<TO, E>(a, s, s.tiles);
    const uint32_t i0 = blockIdx.x * kSortTile + warp * (32 * kSortRounds) + lane;
    uint32_t key[kSortRounds], pos[kSortRounds], rank[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const uint32_t i = i0 + r * 32;
        key[r] = i < a.n ? sort_key(a, s, i) : 0;
        pos[r] = i < a.n ? (s.first ? i : s.pos_in[i]) : 0;
    }
    // two digits a thread: pairs of smaller digits, of this digit in tiles before
    const uint32_t d0 = tid * 2;
    uint32_t total[2] = {0, 0}, before[2] = {0, 0};
    if (s.totals) {
        for (int k = 0; k < 2; ++k) {
            total[k] = s.totals[d0 + k];
            before[k] = s.counts[size_t(blockIdx.x) * kDigits + d0 + k];
        }
    } else {
        const uint32_t group = blockIdx.x / kGroup, groups = (s.tiles + kGroup - 1) / kGroup;
        // (a fixed number of reads at a time, all on their way at once, those outside left out)
        for (uint32_t g0 = 0; g0 < groups; g0 += kAtOnce) {
            uint2 c[kAtOnce];
#pragma unroll
            for (uint32_t i = 0; i < kAtOnce; ++i)
                c[i] = g0 + i < groups ? reinterpret_cast<const uint2*>(s.groups)[size_t(g0 + i) * (kDigits / 2) + tid] : make_uint2(0, 0);
#pragma unroll
            for (uint32_t i = 0; i < kAtOnce; ++i) {
                total[0] += c[i].x;
                total[1] += c[i].y;
                before[0] += g0 + i < group ? c[i].x : 0;
                before[1] += g0 + i < group ? c[i].y : 0;
            }
        }
        uint2 c[kGroup - 1];
#pragma unroll
        for (uint32_t i = 0; i < kGroup - 1; ++i) {
            const uint32_t t = group * kGroup + i;
            c[i] = t < blockIdx.x ? reinterpret_cast<const uint2*>(s.counts)[size_t(t) * (kDigits / 2) + tid] : make_uint2(0, 0);
        }
#pragma unroll
        for (uint32_t i = 0; i < kGroup - 1; ++i) {
            before[0] += c[i].x;
            before[1] += c[i].y;
        }
    }
    for (uint32_t d = tid; d < kSortWarps * kDigits; d += kSortThreads) (&count[0][0])[d] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const bool there = i0 + r * 32 < a.n;
        const uint32_t d = (key[r] >> s.shift) & (kDigits - 1), same = same_digit(d, there);
        rank[r] = there ? count[warp][d] + __popc(same & ((1u << lane) - 1)) : 0;
        __syncwarp();
        if (there && lane == uint32_t(__ffs(same) - 1)) count[warp][d] += __popc(same);
        __syncwarp();
    }
    uint32_t scan = total[0] + total[1];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint32_t up = __shfl_up_sync(kFull, scan, o);
        if (lane >= uint32_t(o)) scan += up;
    }
    if (lane == 31) warp_sum[warp] = scan;
    __syncthreads();
    uint32_t base = scan - total[0] - total[1];
    for (uint32_t w = 0; w < warp; ++w) base += warp_sum[w];
    uint32_t at[2] = {base + before[0], base + total[0] + before[1]};
#pragma unroll
    for (int k = 0; k < 2; ++k)
        for (int w = 0; w < kSortWarps; ++w) {
            const uint32_t c = count[w][d0 + k];
            count[w][d0 + k] = at[k];
            at[k] += c;
        }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r)
        if (i0 + r * 32 < a.n) {
            const uint32_t to = count[warp][(key[r] >> s.shift) & (kDigits - 1)] + rank[r];
            s.key_out[to] = key[r];
            s.pos_out[to] = pos[r];
            if (!s.last) {
                const uint32_t d = (key[r] >> (s.shift + kDigitBits)) & (kDigits - 1);
                atomicAdd(&s.next_counts[size_t(to / kSortTile) * kDigits + d], 1u);
                atomicAdd(&s.next_groups[size_t(to / kSortTile / kGroup) * kDigits + d], 1u);
            }
        }
}

// Where runs of equal ids begin and end
template <class TO, int E>
__global__ void __launch_bounds__(kSortThreads) mark_runs_kernel(GradArgs a, SortArgs s) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t marks = (a.n + kSortThreads - 1) / kSortThreads;
    if (blockIdx.x >= marks) return clear_unnamed<TO, E>(a, s, marks);
    const uint32_t i = blockIdx.x * kSortThreads + threadIdx.x;
    if (i >= a.n) return;
    const uint32_t k = a.key[i];
    if (k == a.rows) return;
    if (i + 1 == a.n || a.key[i + 1] != k) a.range[k].y = i + 1;
    if (i == 0 || a.key[i - 1] != k) a.range[k].x = i;
}

// A warp sums 32 vectors of the rows of `grad` that places name, in the places' order: those of `todo` lanes from
// `first` on.  At the lanes in `fresh` a run begins: `changed` is called with its lane before its sum.  Rows come by asynchronous copies, kDepth of them on their
// way, each lane its own bytes to its own place.  (By loads, four rows at a time: 131,072 tokens of 1,024 bf16 values 84 us
// instead of 64 to 66.)
constexpr int kSumThreads = 256, kDepth = 8;

template <class T, int E>
__device__ __forceinline__ void copy_vector(Pack<T, E>* to, const T* from) {
    if constexpr (Pack<T, E>::kBytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
    else if constexpr (Pack<T, E>::kBytes >= 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(to)), "l"(from), "n"(Pack<T, E>::kBytes) : "memory");
    else
        to->load(from);
}

template <class TI, int E, class F>
__device__ __forceinline__ void sum_rows(const GradArgs& a, uint32_t first, uint32_t todo, uint32_t fresh, uint32_t pos, uint32_t v, bool inside, Pack<TI, E>* ring,
                                         float (&sum)[E], F changed) {
    const TI* grad = static_cast<const TI*>(a.grad) + size_t(v) * E;
    uint32_t asked = 0;
    auto ask = [&](int slot) {
        if (asked < todo) {
            const uint32_t p = __shfl_sync(kFull, pos, first + asked++);
            if (inside) copy_vector<TI, E>(ring + slot * 32, grad + p * a.grad_stride);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int k = 0; k < kDepth; ++k) ask(k);
    for (uint32_t done = 0; done < todo;) {
#pragma unroll
        for (int k = 0; k < kDepth; ++k) {
            if (done == todo) break;
            if (fresh >> (first + done) & 1) changed(first + done);
            ++done;
            asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
            Pack<TI, E> x = ring[k * 32];
            ask(k);
            if constexpr (E >= 2) {
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const Two t = add({sum[e], sum[e + 1]}, {x.get(e), x.get(e + 1)});
                    sum[e] = t.x;
                    sum[e + 1] = t.y;
                }
            } else {
                sum[0] += x.get(0);
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// A warp takes the runs that begin among its kEntries places of the sorted pairs, to their ends.  (A warp for each row of the
// output, with the row's range to read, then its places, then their rows, waited for one load after the other: 131,072 tokens
// of 1,024 bf16 values 160 us.)
// The first blocks take the pieces of long runs instead.
constexpr uint32_t kEntries = 16;

// Piece p of the run `r` of row k, as a warp has summed 32 vectors of it: the warp that brings the last of kJoin pieces adds
// them up, in their order, the one that brings the last of kJoin such sums adds those up, and so on.  Who does it depends on
// the time, the result does not.  (A launch of its own for it took 10 us for the 161 longest runs of 131,072 tokens; here it
// goes on beside other sums.)
template <class TO, int E>
__device__ __forceinline__ void join_piece(const GradArgs& a, uint32_t k, uint2 r, uint32_t p, uint32_t v, bool inside, float (&sum)[E]) {
    const uint32_t c0 = r.x / kRun, pieces = (r.y - 1) / kRun - c0 + 1;
    auto at = [&](uint32_t piece) { return size_t(c0 + piece) * 2 + (piece == 0 && r.x % kRun != 0); };
    auto store = [&](uint32_t piece) {
        Pack<float, E> o;
#pragma unroll
        for (int e = 0; e < E; ++e) o.set(e, sum[e]);
        if (inside) o.store(a.partial + at(piece) * a.dim + size_t(v) * E);
    };
    // whether all of `many` are there, this one the last
    auto arrive = [&](uint32_t* counter, uint32_t many) {
        __threadfence();
        __syncwarp();
        uint32_t before = 0;
        if ((threadIdx.x & 31) == 0) before = atomicAdd(counter, 1u);
        const bool last = __shfl_sync(kFull, before, 0) + 1 == many;
        if (last) __threadfence();
        return last;
    };
    auto add_up = [&](uint32_t first, uint32_t step, uint32_t many) {
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] = 0.0f;
        if (!inside) return;
#pragma unroll 4
        for (uint32_t i = 0; i < many; ++i) {
            Pack<float, E> x;  // (from L2: other SMs have written it)
            const typename Pack<float, E>::Raw* from = reinterpret_cast<const typename Pack<float, E>::Raw*>(a.partial + at(first + i * step) * a.dim + size_t(v) * E);
#pragma unroll
            for (int w = 0; w < Pack<float, E>::kWords; ++w) x.raw[w] = __ldcg(from + w);
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] += x.get(e);
        }
    };
    const size_t counters = (size_t(a.n) / kRun + 1) * 2 * a.parts;
    uint32_t step = 1, left = pieces;  // what is joined: every step-th piece's place, `left` in all
#pragma unroll 1
    for (int level = 0;; ++level) {
        store(p * step);
        const bool top = level == kJoinLevels - 1;
        const uint32_t first = top ? 0 : p / kJoin * kJoin, many = top ? left : min(kJoin, left - first);
        if (!arrive(a.arrived + counters * level + at(first * step) * a.parts + v / 32, many)) return;
        add_up(first * step, step, many);
        if (many == left) break;
        p /= kJoin;
        step *= kJoin;
        left = (left + kJoin - 1) / kJoin;
    }
    if (inside) write_sum<TO, E>(a, static_cast<TO*>(a.out) + k * a.out_stride + size_t(v) * E, sum);
}

template <class TI, class TO, int E>
__global__ void __launch_bounds__(kSumThreads) grad_sums_kernel(GradArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ __align__(16) unsigned char ring_smem[kSumThreads * kDepth * sizeof(Pack<TI, E>)];
    const int lane = threadIdx.x & 31;
    Pack<TI, E>* mine_ring = reinterpret_cast<Pack<TI, E>*>(ring_smem) + (threadIdx.x >> 5) * (kDepth * 32) + lane;
    const uint32_t vecs = a.dim / E;
    float sum[E];
    auto clear = [&] {
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] = 0.0f;
    };
    if (blockIdx.x < a.piece_blocks) {
        // piece `c` of the sorted pairs: what it holds of the long run that covers its first place, and of the one that
        // covers its last place and begins inside
        const uint64_t item = (uint64_t(blockIdx.x) * kSumThreads + threadIdx.x) >> 5;
        const uint32_t c = uint32_t(item / a.parts), v = uint32_t(item % a.parts) * 32 + lane;
        const bool inside = v < vecs;
        if (uint64_t(c) * kRun >= a.n) return;
        const uint32_t from = c * kRun, to = min(a.n, from + kRun);
        const uint32_t k0 = a.key[from], k1 = a.key[to - 1];
#pragma unroll 1
        for (int side = 0; side < 2; ++side) {
            const uint32_t k = side ? k1 : k0;
            if (k == a.rows || (side && k1 == k0)) continue;
            const uint2 r = a.range[k];
            if (r.y - r.x <= kRun) continue;
            const uint32_t first = max(from, r.x), end = min(to, r.y);
            clear();
            for (uint32_t base = first; base < end; base += 32) {
                const bool there = base + lane < end;
                sum_rows<TI, E>(a, 0, min(32u, end - base), 0u, there ? a.pos[base + lane] : 0, v, inside, mine_ring, sum, [](uint32_t) {});
            }
            join_piece<TO, E>(a, k, r, c - r.x / kRun, v, inside, sum);
        }
        return;
    }
    const uint64_t item = (uint64_t(blockIdx.x - a.piece_blocks) * kSumThreads + threadIdx.x) >> 5;
    const uint64_t i0 = item / a.parts * kEntries;
    if (i0 >= a.n) return;
    const uint32_t v = uint32_t(item % a.parts) * 32 + lane;
    const bool inside = v < vecs;
    TO* out = static_cast<TO*>(a.out) + size_t(v) * E;
    uint32_t row = a.rows;  // whose sum is held; rows: none
    auto flush = [&] {
        if (row != a.rows && inside) write_sum<TO, E>(a, out + row * a.out_stride, sum);
        clear();
    };
    clear();
    for (uint64_t base = i0;; base += 32) {
        const uint64_t i = base + lane;
        const bool there = i < a.n, own = base == i0;  // own: runs may begin here
        const uint32_t key = there ? a.key[i] : a.rows, pos = there ? a.pos[i] : 0;
        const uint32_t before = there && i > 0 ? a.key[i - 1] : a.rows + 1;
        const uint32_t after = own && i + kRun < a.n ? a.key[i + kRun] : a.rows;
        const uint32_t starts = __ballot_sync(kFull, key != before || !there);
        // the place where this one's run begins: among these, or earlier
        const uint32_t upto = starts & (0xffffffffu >> (31 - lane));
        const int start = upto ? 31 - __clz(upto) : -1;
        const bool long_run = __shfl_sync(kFull, int(key != a.rows && after == key), start < 0 ? 0 : start);
        const bool mine = key != a.rows && (own ? start >= 0 && start < int(kEntries) && !long_run : start < 0 && key == row);
        // (these lanes are neighbours: a run longer than kRun, or of no row, goes on behind the last of them)
        static_assert(kRun >= 32, "else a long run could end among these places");
        const uint32_t summed = __ballot_sync(kFull, mine);
        sum_rows<TI, E>(a, summed ? __ffs(summed) - 1 : 0, __popc(summed), starts, pos, v, inside, mine_ring, sum, [&](uint32_t at) {
            flush();
            row = __shfl_sync(kFull, key, at);
        });
        // the last run may go on behind these places
        const uint32_t last = __shfl_sync(kFull, key, 31);
        if (row == a.rows || last != row) break;
    }
    flush();
}

// Workspace of the sorted form, in bytes from its start; what has to be zero at the start comes first
struct GradSpace {
    uint64_t tiles;
    int passes;
    size_t named, counts, groups, arrived, totals, key[2], pos[2], range, partial, bytes;
    static uint64_t join_counters(uint64_t n, uint64_t parts) { return (n / kRun + 1) * 2 * parts; }
    GradSpace(uint64_t n, uint64_t rows, uint64_t dim) {
        size_t at = 0;
        auto take = [&](size_t b) {
            const size_t here = at;
            at += (b + 255) / 256 * 256;
            return here;
        };
        tiles = (n + kSortTile - 1) / kSortTile;
        passes = 0;
        while (rows >> (passes * kDigitBits)) ++passes;  // (`rows` itself is the key of an id that is none)
        named = take(rows * 4);
        counts = take(passes * tiles * kDigits * 4);
        groups = take(passes * (tiles / kGroup + 1) * kDigits * 4);
        arrived = take(kJoinLevels * join_counters(n, (dim + 31) / 32) * 4);  // (parts are fewer where accesses are of several elements)
        totals = take(kDigits * 4);
        for (int i = 0; i < 2; ++i) key[i] = take(n * 4), pos[i] = take(n * 4);
        range = take(rows * 8);
        partial = take((n / kRun + 1) * 2 * dim * 4);
        bytes = at;
    }
};

// A launch that may begin while the kernel in front of it ends, and waits for that by itself
template <class... P, class... Q>
int launch_behind(void (*kernel)(P...), dim3 grid, int threads, cudaStream_t st, const Q&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    CPB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    return 0;
}

template <class TI, class TO, int E>
int launch_grad(GradArgs& a, void* workspace, cudaStream_t st) {
    const uint32_t vecs = a.dim / E;
    if (a.n <= kSmallMost) {
        const uint64_t clear = a.accumulate ? 0 : (uint64_t(a.rows) + kClearRows - 1) / kClearRows;
        // As many groups as there are where a thread has one vector of the most values that the row's length allows.  What the layouts
        // leave of that (E) changes how many vectors a thread takes, not the groups, so that the order of a sum does not depend on
        // where rows start.  (300 places of 15 ids, 512 bf16 values: 5.0 us; from rows at odd addresses 16.5, and 14 with as many groups
        // as E would have.)
        uint32_t most = 16 / sizeof(TI), along = 32;
        while (a.dim % most) most /= 2;
        while (along < a.dim / most && along < kSmallThreads) along *= 2;
        a.most_groups = kSmallThreads / along;
        if (a.n + clear) grad_small_kernel<TI, TO, E><<<unsigned(a.n + clear), kSmallThreads, 0, st>>>(a);
        CPB_CUDA(cudaGetLastError());
        return 0;
    }
    const GradSpace at(a.n, a.rows, a.dim);
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    a.range = reinterpret_cast<uint2*>(ws + at.range);
    a.arrived = reinterpret_cast<uint32_t*>(ws + at.arrived);
    a.parts = (vecs + 31) / 32;
    const uint64_t counters = kJoinLevels * GradSpace::join_counters(a.n, a.parts);
    a.partial = reinterpret_cast<float*>(ws + at.partial);
    CPB_CUDA(cudaMemsetAsync(ws, 0, at.arrived + counters * 4, st));
    SortArgs s{};
    s.tiles = uint32_t(at.tiles);
    s.named = reinterpret_cast<uint32_t*>(ws + at.named);
    s.counts = reinterpret_cast<uint32_t*>(ws + at.counts);
    s.groups = reinterpret_cast<uint32_t*>(ws + at.groups);
    s.first = 1;
    sort_count_kernel<<<s.tiles, kSortThreads, 0, st>>>(a, s);
    CPB_CUDA(cudaGetLastError());
    // the rows to clear, in equal parts beside the passes and the marks
    auto part = [&](int k) { return uint64_t(a.rows) * k / (at.passes + 1); };
    auto clear_blocks = [&](int k) {
        if (a.accumulate) return uint64_t(0);
        s.clear0 = part(k);
        s.clear1 = part(k + 1);
        constexpr uint64_t kRows = kSortThreads / 32 * kClearWarpRows;  // of a block
        return (s.clear1 - s.clear0 + kRows - 1) / kRows;
    };
    for (int pass = 0; pass < at.passes; ++pass) {
        s.shift = pass * kDigitBits;
        s.first = pass == 0;
        s.last = pass + 1 == at.passes;
        s.next_counts = s.counts + size_t(s.tiles) * kDigits;
        s.next_groups = s.groups + size_t(s.tiles / kGroup + 1) * kDigits;
        s.key_in = reinterpret_cast<uint32_t*>(ws + at.key[(pass & 1) ^ 1]);
        s.pos_in = reinterpret_cast<uint32_t*>(ws + at.pos[(pass & 1) ^ 1]);
        s.key_out = reinterpret_cast<uint32_t*>(ws + at.key[pass & 1]);
        s.pos_out = reinterpret_cast<uint32_t*>(ws + at.pos[pass & 1]);
        if (s.tiles > kFoldTiles) {
            s.totals = reinterpret_cast<uint32_t*>(ws + at.totals);
            CPB_TRY(launch_behind(sort_scan_kernel, dim3(kDigits / 32), 1024, st, s.counts, s.totals, s.tiles));
        }
        const uint64_t blocks = s.tiles + clear_blocks(pass);
        CPB_TRY(launch_behind(sort_place_kernel<TO, E>, dim3(unsigned(blocks)), kSortThreads, st, a, s));
        s.counts = s.next_counts;
        s.groups = s.next_groups;
    }
    a.key = s.key_out;
    a.pos = s.pos_out;
    const uint64_t blocks = (a.n + kSortThreads - 1) / kSortThreads + clear_blocks(at.passes);
    CPB_TRY(launch_behind(mark_runs_kernel<TO, E>, dim3(unsigned(blocks)), kSortThreads, st, a, s));
    constexpr uint64_t kWarps = kSumThreads / 32;
    const uint64_t pieces = (uint64_t(a.n) + kRun - 1) / kRun, entries = (uint64_t(a.n) + kEntries - 1) / kEntries;
    const uint64_t piece_blocks = (pieces * a.parts + kWarps - 1) / kWarps, entry_blocks = (entries * a.parts + kWarps - 1) / kWarps;
    CPB_OP_CHECK(piece_blocks + entry_blocks < (1ull << 31), "embedding_grad: too many places for one call");
    a.piece_blocks = uint32_t(piece_blocks);
    return launch_behind(grad_sums_kernel<TI, TO, E>, dim3(unsigned(piece_blocks + entry_blocks)), kSumThreads, st, a);
}

template <class TI, class TO>
int pick_grad(GradArgs& a, void* ws, cudaStream_t st) {
    // E elements, a divisor of the row: up to 16 bytes of `grad` by one load and all of them to `out` by one store, which for eight
    // sums of fp32 is one of 32 bytes; either side's rows start at multiples of the access
    auto fits = [&](uint32_t e) {
        const uint64_t in = e * sizeof(TI) < 16 ? e * sizeof(TI) : 16, out = e * sizeof(TO);
        Alignment i, o;
        i.add(a.grad).add(a.grad_stride * sizeof(TI));
        o.add(a.out).add(a.out_stride * sizeof(TO));
        return a.dim % e == 0 && i.holds(in) && o.holds(out);
    };
    if (sizeof(TI) == 2 && fits(8)) return launch_grad<TI, TO, sizeof(TI) == 2 ? 8 : 4>(a, ws, st);
    if (fits(4)) return launch_grad<TI, TO, 4>(a, ws, st);
    if (fits(2)) return launch_grad<TI, TO, 2>(a, ws, st);
    return launch_grad<TI, TO, 1>(a, ws, st);
}

}  // namespace
}  // namespace cpb

using namespace cpb;

extern "C" {

int cphnsw_b200_embedding_lookup_dev(const void* d_table, int type, uint64_t rows, uint64_t dim, uint64_t table_stride,
                                     const void* d_ids, uint32_t id_bytes, uint64_t n, float scale, void* d_out,
                                     uint64_t out_stride, void* stream) {
    CPB_OP_CHECK(op::type_known(type), "embedding_lookup: unknown element type");
    CPB_OP_CHECK(id_bytes == 4 || id_bytes == 8, "embedding_lookup: ids have 4 or 8 bytes");
    CPB_OP_CHECK(rows >= 1 && rows < (1ull << 31), "embedding_lookup: need 1 <= rows < 2^31");
    CPB_OP_CHECK(dim >= 1 && dim < (1ull << 31), "embedding_lookup: need 1 <= dim < 2^31");
    CPB_OP_CHECK(out_stride >= dim || n <= 1, "embedding_lookup: rows of the output overlap");
    if (n == 0) return 0;
    CPB_OP_CHECK(n < (1ull << 40), "embedding_lookup: too many rows for one call");
    CPB_OP_CHECK(d_table && d_ids && d_out, "embedding_lookup: null pointer");
    CPB_OP_CHECK(op::Alignment().add(d_table).add(d_out).holds(op::type_bytes(type)) && op::Alignment().add(d_ids).holds(id_bytes),
                 "embedding_lookup: an address is no multiple of its element's size");
    CPB_TRY(op::check_device());
    LookupArgs a{};
    a.table = d_table;
    a.out = d_out;
    a.ids = {d_ids, id_bytes, uint32_t(rows)};
    a.n = n;
    a.table_stride = table_stride;
    a.out_stride = out_stride;
    a.dim = uint32_t(dim);
    a.scale = scale;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (type) {
        case CPHNSW_B200_F32: return pick_lookup<float>(a, st);
        case CPHNSW_B200_F16: return pick_lookup<__half>(a, st);
        default: return pick_lookup<__nv_bfloat16>(a, st);
    }
}

uint64_t cphnsw_b200_embedding_grad_workspace(uint64_t n, uint64_t rows, uint64_t dim) {
    // (what the call refuses needs none; the digits of `rows` are counted by shifts of it)
    if (n <= kSmallMost || n >= (1ull << 31) || rows >= (1ull << 31) || dim >= (1ull << 20)) return 0;
    return GradSpace(n, rows, dim).bytes;
}

int cphnsw_b200_embedding_grad_dev(const void* d_ids, uint32_t id_bytes, uint64_t n, const void* d_grad, int grad_type,
                                   uint64_t grad_stride, float scale, void* d_out, int out_type, uint64_t rows, uint64_t dim,
                                   uint64_t out_stride, int accumulate, void* d_workspace, uint64_t workspace_bytes,
                                   void* stream) {
    CPB_OP_CHECK(op::type_known(grad_type) && (out_type == grad_type || out_type == CPHNSW_B200_F32),
                 "embedding_grad: the output has the gradient's type or fp32");
    CPB_OP_CHECK(id_bytes == 4 || id_bytes == 8, "embedding_grad: ids have 4 or 8 bytes");
    CPB_OP_CHECK(rows >= 1 && rows < (1ull << 31), "embedding_grad: need 1 <= rows < 2^31");
    CPB_OP_CHECK(dim >= 1 && dim < (1ull << 20), "embedding_grad: need 1 <= dim < 2^20");
    CPB_OP_CHECK(n < (1ull << 31), "embedding_grad: need n < 2^31");
    CPB_OP_CHECK(out_stride >= dim || rows == 1, "embedding_grad: rows of the output overlap");
    CPB_OP_CHECK(d_out && (n == 0 || (d_ids && d_grad)), "embedding_grad: null pointer");
    CPB_OP_CHECK(op::Alignment().add(d_grad).holds(op::type_bytes(grad_type)) && op::Alignment().add(d_out).holds(op::type_bytes(out_type)) &&
                     op::Alignment().add(d_ids).holds(id_bytes),
                 "embedding_grad: an address is no multiple of its element's size");
    const uint64_t need = cphnsw_b200_embedding_grad_workspace(n, rows, dim);
    CPB_OP_CHECK(workspace_bytes >= need && (need == 0 || (d_workspace && op::Alignment().add(d_workspace).holds(256))),
                 "embedding_grad: the workspace is too small, or not aligned to 256 bytes");
    CPB_TRY(op::check_device());
    GradArgs a{};
    a.ids = {d_ids, id_bytes, uint32_t(rows)};
    a.grad = d_grad;
    a.out = d_out;
    a.grad_stride = grad_stride;
    a.out_stride = out_stride;
    a.n = uint32_t(n);
    a.rows = uint32_t(rows);
    a.dim = uint32_t(dim);
    a.accumulate = accumulate != 0;
    a.scale = scale;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (grad_type) {
        case CPHNSW_B200_F32: return pick_grad<float, float>(a, d_workspace, st);
        case CPHNSW_B200_F16:
            return out_type == CPHNSW_B200_F32 ? pick_grad<__half, float>(a, d_workspace, st) : pick_grad<__half, __half>(a, d_workspace, st);
        default:
            return out_type == CPHNSW_B200_F32 ? pick_grad<__nv_bfloat16, float>(a, d_workspace, st)
                                               : pick_grad<__nv_bfloat16, __nv_bfloat16>(a, d_workspace, st);
    }
}

}  // extern "C"
