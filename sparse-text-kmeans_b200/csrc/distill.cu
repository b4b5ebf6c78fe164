// Distillation from a teacher's top logits: the loss of every row, and its gradient.
//
// A row has the student's logits z_v over all `rows` candidates and a list of the teacher's (id t_j, logit s_j); a place of
// the list whose id lies outside [0, rows) is empty.  With a temperature T,
//   p = softmax(s / T) over the list,   q = softmax(z / T) over all candidates,
//   loss = T^2 sum_j p_j (log p_j - log q_{t_j}),   dz_v = weight T (q_v - sum over j with t_j = v of p_j).
// A row whose list is empty (or all -inf) has loss 0 and gradient 0 whatever z holds; one whose logits are all -inf has
// q = 0 throughout, and a loss of +inf.  Weight 0 gives a gradient of 0 whatever z holds.
// A NaN or +inf among the logits makes the row's loss and all of its gradient NaN, a NaN among the list's the loss and the
// gradient at the list's ids.
//
// Everything is computed in fp32: z_v is read as it is stored, q_v = 2^((z_v - m) c) / sum with c = log2(e) / T and m the
// row's maximum, so that the size of the logits costs no precision; the gradient is rounded to the logits' type once.  A row's
// maximum and sum are joined in a fixed order: thread, warp, block, cluster.
#include "mma_common.cuh"
#include "operators_common.cuh"

namespace cpb {
namespace {

using namespace op;

constexpr int kWords = 8;                 // 16-byte words of a row that a thread takes at a time
constexpr uint32_t kMaxTop = 1024;        // places of a list
constexpr uint32_t kMaxCluster = 8;       // blocks that share a row
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
    const void* z;
    void* grad;            // NULL: the loss alone
    Ids ids;
    const float* teacher;
    const float* weight;   // NULL: 1
    float* loss;
    float2* stats;         // [n] (maximum, sum): written by the loss where not NULL, read where a row goes in pieces
    float4* sums;          // [n] of the lists (ListSums)
    unsigned char* lists;  // [n][top * 12 bytes] (List)
    uint64_t n, z_stride, grad_stride, ids_stride, teacher_stride;  // in elements
    uint32_t rows, top, pieces;
    uint32_t per, slots;   // words of a row that a block has; chunks in its ring
    int ahead;             // rows that some of a block's warps may be ahead of others
    uint32_t* status;
    float T, c;            // c = log2(e) / T
    int same_phase;        // a row of z and its gradient start at the same place of a 16-byte word
};

// 2^x: exact to about 2^-22, results below the smallest normal number are 0
__device__ __forceinline__ float exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// ---- words of a row -----------------------------------------------------------------------------------------------------
// 16 bytes of T: as pairs of fp32, and the larger of two words element by element (a NaN loses: the sums show it)
template <class T>
struct Word;
template <>
struct Word<float> {
    static constexpr uint32_t kNothing = 0xff800000u;  // -inf throughout
    __device__ __forceinline__ static Two pair(const uint4& w, int i) {
        return i ? Two{__uint_as_float(w.z), __uint_as_float(w.w)} : Two{__uint_as_float(w.x), __uint_as_float(w.y)};
    }
    __device__ __forceinline__ static uint32_t max2(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
    __device__ __forceinline__ static float top(uint32_t a) { return __uint_as_float(a); }
};
template <>
struct Word<__half> {
    static constexpr uint32_t kNothing = 0xfc00fc00u;
    __device__ __forceinline__ static Two pair(const uint4& w, int i) {
        const uint32_t u = i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
        return {f.x, f.y};
    }
    __device__ __forceinline__ static uint32_t max2(uint32_t a, uint32_t b) {
        const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    __device__ __forceinline__ static float top(uint32_t a) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a));
        return fmaxf(f.x, f.y);
    }
};
template <>
struct Word<__nv_bfloat16> {
    static constexpr uint32_t kNothing = 0xff80ff80u;
    __device__ __forceinline__ static Two pair(const uint4& w, int i) {
        const uint32_t u = i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
        return {__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)};
    }
    __device__ __forceinline__ static uint32_t max2(uint32_t a, uint32_t b) {
        const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    __device__ __forceinline__ static float top(uint32_t a) { return fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u)); }
};
template <class T>
__device__ __forceinline__ uint4 nothing() {
    return make_uint4(Word<T>::kNothing, Word<T>::kNothing, Word<T>::kNothing, Word<T>::kNothing);
}
template <class T, int W>
__device__ __forceinline__ float max_of(const uint4 (&w)[W]) {
    uint4 m = w[0];
#pragma unroll
    for (int j = 1; j < W; ++j)
        m = make_uint4(Word<T>::max2(m.x, w[j].x), Word<T>::max2(m.y, w[j].y), Word<T>::max2(m.z, w[j].z), Word<T>::max2(m.w, w[j].w));
    return Word<T>::top(Word<T>::max2(Word<T>::max2(m.x, m.y), Word<T>::max2(m.z, m.w)));
}
// What is subtracted from a logit before it is scaled: the maximum, or 0 of a row that is -inf throughout.  (Scaling first,
// to use one fused operation, is off by the rounding of m c: of a row at its type's lowest value nothing would be left.)
__device__ __forceinline__ float shift_of(float m) { return m == -INFINITY ? 0.0f : m; }
template <class T>
__device__ __forceinline__ void add_word(Two& sum, const uint4& w, Two away, Two scale) {
#pragma unroll
    for (int i = 0; i < int(8 / sizeof(T)); ++i) {
        const Two x = mul(add(Word<T>::pair(w, i), away), scale);
        sum = add(sum, {exp2(x.x), exp2(x.y)});
    }
}
template <class T, int W>
__device__ __forceinline__ float sum_of(const uint4 (&w)[W], float m, float c) {
    const Two away{-shift_of(m), -shift_of(m)}, scale{c, c};
    Two sum{0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < W; ++j) add_word<T>(sum, w[j], away, scale);
    return sum.x + sum.y;
}

template <class T>
struct Row {
    static constexpr int E = 16 / int(sizeof(T));
    const T* p;      // first logit
    uint32_t head;   // elements of the first 128-byte line that lie before it: words count from the line's start
    uint32_t words;
    __device__ __forceinline__ Row(const void* base, uint64_t row, uint64_t stride, uint32_t rows) {
        p = static_cast<const T*>(base) + row * stride;
        head = uint32_t(reinterpret_cast<uintptr_t>(p) & 127) / sizeof(T);
        words = uint32_t((uint64_t(head) + rows + E - 1) / E);
    }
    // word w; elements outside the row are -inf and are not read
    __device__ __forceinline__ uint4 load(uint32_t w, uint32_t rows) const {
        const int64_t col = int64_t(w) * E - head;
        if (col >= 0 && col + E <= int64_t(rows)) return __ldcs(reinterpret_cast<const uint4*>(p + col));
        Pack<T, E> x;
        x.raw[0] = nothing<T>();
        if (w < words) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (col + e >= 0 && col + e < int64_t(rows)) x.v[e] = p[col + e];
        }
        return x.raw[0];
    }
};
template <class T>
__device__ __forceinline__ void write_word(T* out, int64_t col, uint32_t rows, bool whole, const uint4& word) {
    constexpr int E = Row<T>::E;
    if (whole && col >= 0 && col + E <= int64_t(rows)) {
        __stcs(reinterpret_cast<uint4*>(out + col), word);
    } else {
        Pack<T, E> x;
        x.raw[0] = word;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (col + e >= 0 && col + e < int64_t(rows)) out[col + e] = x.v[e];
    }
}

// ---- a maximum and the sum of 2^((z - maximum) c) ---------------------------------------------------------------------------
struct MaxSum {
    float m = -INFINITY, s = 0.0f;
};
// s taken from the maximum m to `to`, which is at least m
__device__ __forceinline__ float moved(float s, float m, float to, float c) { return m == to || s == 0.0f ? s : s * exp2((m - to) * c); }

// ---- cluster --------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait;" ::: "memory"); }
__device__ __forceinline__ void store_to_block(float* smem, uint32_t rank, float v) {
    uint32_t addr;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(smem)), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// ---- block ----------------------------------------------------------------------------------------------------------------
struct List {
    float* p;                // [top] the teacher's probabilities
    float* z;                // [top] the student's logits at the list's ids
    uint32_t* id;            // [top]
    __device__ __forceinline__ List(void* at, uint32_t top) {
        p = static_cast<float*>(at);
        z = p + top;
        id = reinterpret_cast<uint32_t*>(z + top);
    }
};
__host__ __device__ constexpr uint32_t list_bytes(uint32_t top) { return top * 12; }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
    return v;
}

// What the loss takes from a row's list besides the row's maximum and sum: sums of p_j log p_j, p_j (z_j - ref) and p_j,
// ref one of the z_j.  p is 0 where nothing in the list counts, and near 1 else.
struct ListSums {
    float plogp, pz, p, ref;
};
// By a warp: the list's ids (kFull where a place is empty), probabilities, and the student's logits there.
template <class T>
__device__ __forceinline__ ListSums read_list(const Args& a, uint64_t row, const List& list) {
    const uint32_t lane = threadIdx.x & 31;
    const T* z = static_cast<const T*>(a.z) + row * a.z_stride;
    float best = -INFINITY, ref = -INFINITY;
    bool any = false;
    // (kAtOnce places a lane on their way together: one after the other, the lists of 1,021 rows, 100 places
    // each, took 16 us instead of 11)
    constexpr int kAtOnce = 4;
    for (uint32_t j0 = lane; j0 < a.top; j0 += 32 * kAtOnce) {
        uint32_t id[kAtOnce];
        float s[kAtOnce], zj[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const uint32_t j = j0 + k * 32;
            id[k] = j < a.top ? a.ids.at(row * a.ids_stride + j) : kFull;
            s[k] = j < a.top ? __ldg(a.teacher + row * a.teacher_stride + j) : -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            if (s[k] == -INFINITY) id[k] = kFull;  // (a NaN counts: the loss is NaN, and the gradient at the list's ids)
            zj[k] = id[k] != kFull ? to_float(z[id[k]]) : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const uint32_t j = j0 + k * 32;
            if (j >= a.top) break;
            if (id[k] != kFull) {
                ref = fmaxf(ref, zj[k]);
                best = fmaxf(best, s[k]);
                any = true;
            }
            list.id[j] = id[k];
            list.p[j] = s[k];
            list.z[j] = zj[k];
        }
    }
    ListSums r{0.0f, 0.0f, 0.0f, 0.0f};
    if (!__any_sync(kFull, any)) return r;
    best = warp_max(best);
    r.ref = shift_of(warp_max(ref));
    float total = 0.0f;
    for (uint32_t j = lane; j < a.top; j += 32)
        if (list.id[j] != kFull) total += exp2((list.p[j] - best) * a.c);
    total = warp_sum(total);
    const float log_total = logf(total), inv_T = 1.0f / a.T, inv_total = 1.0f / total;
    for (uint32_t j = lane; j < a.top; j += 32) {
        const float d = list.p[j] - best, p = list.id[j] == kFull ? 0.0f : exp2(d * a.c) * inv_total;
        list.p[j] = p;
        if (p != 0.0f) {  // (0 log 0 is 0, and so is 0 times a logit of -inf)
            r.plogp += p * (d * inv_T - log_total);
            r.pz += p * (list.z[j] - r.ref);
            r.p += p;
        }
    }
    r.plogp = warp_sum(r.plogp);
    r.pz = warp_sum(r.pz);
    r.p = warp_sum(r.p);
    return r;
}

// Ids that come more than once: the first place takes all their probabilities, in the places' order, the others become
// empty.  By a warp, on a list in shared memory; `table` has table_words(top) words.
__host__ __device__ constexpr uint32_t table_words(uint32_t top) {
    uint32_t n = 64;
    while (n < 2 * top) n *= 2;
    return n;
}
__device__ __forceinline__ void join_repeats(uint32_t top, const List& list, uint32_t* table) {
    const uint32_t lane = threadIdx.x & 31, size = table_words(top);
    for (uint32_t i = lane; i < size; i += 32) table[i] = kFull;
    __syncwarp();
    bool again = false;
    for (uint32_t j = lane; j < top; j += 32) {
        const uint32_t id = list.id[j];
        if (id == kFull) continue;
        // (ids at equal distances, as from a stride, must not meet in a few places: one multiplication is not enough)
        uint32_t at = (id ^ id >> 15) * 0x9e3779b1u;
        at = (at ^ at >> 13) * 0x85ebca6bu;
        for (at = (at ^ at >> 16) & (size - 1);; at = (at + 1) & (size - 1)) {  // (half of the table is empty)
            const uint32_t was = atomicCAS(&table[at], kFull, id);
            again |= was == id;
            if (was == kFull || was == id) break;
        }
    }
    if (!__any_sync(kFull, again)) return;
    for (uint32_t j0 = 0; j0 < top; j0 += 32) {
        const uint32_t j = j0 + lane, id = j < top ? list.id[j] : kFull;
        bool first = true;
        float p = 0.0f;
        for (uint32_t k = 0; k < top && id != kFull; ++k)
            if (list.id[k] == id) {
                first = first && k >= j;
                p += k >= j ? list.p[k] : 0.0f;
            }
        __syncwarp();  // (places behind these are as they were; of those before, the first of an id still has it)
        if (id != kFull) {
            if (first)
                list.p[j] = p;
            else
                list.id[j] = kFull;
        }
        __syncwarp();
    }
}

__device__ __forceinline__ float loss_of(const Args& a, const ListSums& l, const MaxSum& r) {
    if (l.p == 0.0f) return 0.0f;  // nothing in the list counts
    const float log_sum = r.s == 0.0f ? 0.0f : logf(r.s);
    return a.T * a.T * (l.plogp - (l.pz + l.p * (l.ref - shift_of(r.m))) / a.T + l.p * log_sum);
}

// ---- the loss alone: a cluster of blocks streams a row -----------------------------------------------------------------------
// Reads every logit once, with the running maximum and sum of the softmax; the list's logits are gathered meanwhile.
template <class T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) distill_loss_kernel(Args a) {
    extern __shared__ __align__(16) unsigned char list_smem[];
    __shared__ float of_warp[kThreads / 32][2], of_block[kMaxCluster][2];
    const uint32_t size = cluster_size(), rank = cluster_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t row = blockIdx.x / size;
    const Row<T> z(a.z, row, a.z_stride, a.rows);
    if (size > 1) cluster_arrive_relaxed();
    const uint32_t per = (z.words + size - 1) / size, w0 = min(z.words, rank * per), w1 = min(z.words, w0 + per);
    uint4 x[kWords];
    auto fetch = [&](uint32_t base) {
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
            const uint32_t w = base + j * kThreads + threadIdx.x;
            x[j] = w < w1 ? z.load(w, a.rows) : nothing<T>();
        }
    };
    fetch(w0);
    ListSums list{};
    if (warp == 0 && rank == 0) list = read_list<T>(a, row, List(list_smem, a.top));
    MaxSum acc;
    for (uint32_t base = w0; base < w1;) {
        const float top = fmaxf(acc.m, max_of<T>(x));
        acc.s = moved(acc.s, acc.m, top, a.c) + sum_of<T>(x, top, a.c);
        acc.m = top;
        base += kThreads * kWords;
        if (base < w1) fetch(base);
    }
    const float top = warp_max(acc.m);
    acc.s = warp_sum(moved(acc.s, acc.m, top, a.c));
    if (lane == 0) of_warp[warp][0] = top, of_warp[warp][1] = acc.s;
    __syncthreads();
    auto joined = [&](const float (*parts)[2], uint32_t many) {
        const float m = lane < many ? parts[lane][0] : -INFINITY;
        MaxSum r;
        r.m = warp_max(m);
        r.s = warp_sum(lane < many ? moved(parts[lane][1], m, r.m, a.c) : 0.0f);
        return r;
    };
    if (size > 1) cluster_wait();  // (every block has begun)
    MaxSum r;
    if (warp == 0) r = joined(of_warp, kThreads / 32);
    if (size > 1) {
        if (threadIdx.x == 0) {
            store_to_block(&of_block[rank][0], 0, r.m);
            store_to_block(&of_block[rank][1], 0, r.s);
        }
        cluster_arrive();
        cluster_wait();
        if (warp == 0 && rank == 0) r = joined(of_block, size);
    }
    if (rank == 0 && threadIdx.x == 0) {
        a.loss[row] = loss_of(a, list, r);
        if (a.stats) a.stats[row] = make_float2(r.m, r.s);
    }
}

// ---- loss and gradient of a word --------------------------------------------------------------------------------------------------
struct Factors {
    float shift, factor, taken;  // the gradient is 2^((z - shift) c) factor, less `taken` p_j at the list's ids
    int zero;                    // or all of it 0
    __device__ __forceinline__ Factors() {}
    __device__ __forceinline__ Factors(float T, float weight, const MaxSum& r, bool some) {
        zero = !some || weight == 0.0f;
        shift = shift_of(r.m);
        taken = weight * T;
        factor = r.s == 0.0f ? 0.0f : taken / r.s;
    }
};
template <class T>
__device__ __forceinline__ uint4 gradient_of(const uint4& word, const Factors& f, float c) {
    constexpr int E = 16 / int(sizeof(T));
    const Two away{-f.shift, -f.shift}, scale{c, c}, times{f.factor, f.factor};
    Pack<T, E> g;
    g.raw[0] = make_uint4(0u, 0u, 0u, 0u);
    if (!f.zero) {
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
            const Two e = mul(add(Word<T>::pair(word, k), away), scale);
            const Two q = mul({exp2(e.x), exp2(e.y)}, times);
            g.set2(k, q.x, q.y);
        }
    }
    return g.raw[0];
}

// ---- short rows: a row in the registers of a warp, kHeld words a lane -------------------------------------------------------------
// One read and, for the gradient, one write of the row.
constexpr int kShortWarps = 4;
// Rows are many and each is a chain of waits, so what counts is how many warps an SM holds: as few words a lane as a row needs
// (3, 6, 10 or 16), and registers for that many blocks at the price of a few spills.  8,192 rows of bf16, 64 places a list,
// microseconds in that form, in the next larger one, and without the bound on registers: 600 logits 16, 21, 16; 1,000 logits 19,
// 27, 22; 2,000 logits 29, 43, 39; 4,000 logits 47, -, 52.
constexpr int short_blocks(int held) { return held <= 6 ? 8 : held <= 10 ? 5 : 4; }
template <class T, int kHeld>
__global__ void __launch_bounds__(kShortWarps * 32, short_blocks(kHeld)) distill_short_kernel(Args a) {
    extern __shared__ __align__(16) unsigned char list_smem[];
    constexpr int E = Row<T>::E;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t row = uint64_t(blockIdx.x) * kShortWarps + warp;
    if (row >= a.n) return;
    const Row<T> z(a.z, row, a.z_stride, a.rows);
    T* out = static_cast<T*>(a.grad) + row * a.grad_stride;
    uint4 x[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) x[j] = lane + j * 32 < z.words ? z.load(lane + j * 32, a.rows) : nothing<T>();
    unsigned char* mine = list_smem + warp * (list_bytes(a.top) + table_words(a.top) * 4);
    const List list(mine, a.top);
    const ListSums sums = read_list<T>(a, row, list);
    if (a.grad) join_repeats(a.top, list, reinterpret_cast<uint32_t*>(mine + list_bytes(a.top)));
    MaxSum r;
    r.m = warp_max(max_of<T>(x));
    r.s = warp_sum(sum_of<T>(x, r.m, a.c));
    if (lane == 0) a.loss[row] = loss_of(a, sums, r);
    if (!a.grad) return;
    const Factors f(a.T, a.weight ? __ldg(a.weight + row) : 1.0f, r, sums.p != 0.0f);
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const uint32_t w = lane + j * 32;
        if (w < z.words) write_word<T>(out, int64_t(w) * E - z.head, a.rows, a.same_phase, gradient_of<T>(x[j], f, a.c));
    }
    if (f.zero) return;
    __syncwarp();
    for (uint32_t j = lane; j < a.top; j += 32)
        if (list.id[j] != kFull) out[list.id[j]] = from_float<T>(exp2((list.z[j] - f.shift) * a.c) * f.factor - f.taken * list.p[j]);
}

// ---- both, long rows: a row goes through the shared memory of a cluster once ------------------------------------------------------
// A word to where words do not start
template <class T>
__device__ __noinline__ void store_apart(T* to, uint4 word) {
    Pack<T, Row<T>::E> x;
    x.raw[0] = word;
#pragma unroll
    for (int e = 0; e < Row<T>::E; ++e) to[e] = x.v[e];
}

// The lists of all rows first, a warp each.
constexpr int kListWarps = 4;
template <class T>
__global__ void __launch_bounds__(kListWarps * 32) distill_list_kernel(Args a) {
    extern __shared__ __align__(16) unsigned char list_smem[];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t row = uint64_t(blockIdx.x) * kListWarps + warp;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (the rows' copies and sums need nothing from here)
    if (row >= a.n) return;
    unsigned char* mine = list_smem + warp * (list_bytes(a.top) + table_words(a.top) * 4);
    const List list(mine, a.top);
    const ListSums s = read_list<T>(a, row, list);
    join_repeats(a.top, list, reinterpret_cast<uint32_t*>(mine + list_bytes(a.top)));
    __syncwarp();
    uint32_t* to = reinterpret_cast<uint32_t*>(a.lists + row * list_bytes(a.top));
    for (uint32_t i = lane; i < a.top * 3; i += 32) to[i] = reinterpret_cast<const uint32_t*>(mine)[i];
    if (lane == 0) a.sums[row] = make_float4(s.plogp, s.pz, s.p, s.ref);
}

// A block per SM takes its share of row after row, in chunks of 4 KB through a ring in shared memory that holds more than a
// row's share.  A chunk is a warp's work:
//   copies    four threads ask for chunks as places in the ring come free;
//   sums      warps that take chunks as they arrive, for the maximum and the sum; at the end of the row each sends its own
//             to all blocks of the cluster;
//   lists     one warp that sorts out what of a row's list lies in the share, some rows ahead;
//   rows      one warp that joins a row's maxima and sums and tells the writers what they need; of the cluster's first block
//             it also writes the loss;
//   writes    warps that write the row's chunks' gradients, the list's ids in them last, and free their places.
// So a row's gradient is written while the next rows arrive and are summed.  Logits are read once and gradients written once:
// 8,192 rows of 131,072 bf16 logits 655 us, 6.6 TB/s, which is the memory's rate; 1,021 rows of 100,003 that start anywhere 74
// us (62).  Beside it two exponentials a logit keep their pipe two thirds busy.
// GIVEN: maximum and sum of the row are in a.stats, and blocks take pieces of rows, knowing nothing of one another (rows
// longer than a cluster holds): all warps write.
// kWarps warps sum and as many write: 12 in a block per SM, or, where rows are so short that what is done once a row counts,
// 3 in each of three blocks per SM.
constexpr int ring_threads(int warps) { return (2 * warps + 3) * 32; }
constexpr int ring_blocks(int warps) { return warps == 12 ? 1 : 3; }
constexpr uint32_t kChunkWords = 256, kChunkBytes = kChunkWords * 16;  // 8 words a lane
constexpr int kAhead = 4;         // rows between the first that is summed and the last that is written
// A block sums row i when it has written row i - kAhead, for which all blocks of the cluster have summed that row and so
// written row i - 2 kAhead: what they are sent has this many places.
constexpr int kStats = 2 * kAhead;
constexpr uint32_t kMaxSlots = 52;
constexpr uint32_t kMaxRing = 16;  // blocks that share a row (above eight the device has to be told)

constexpr int kCopiers = 4;       // threads that ask for chunks
// Chunk c of a row, behind `before` chunks of other rows: its place in the ring and its turn there.  A ring has more places
// than a row chunks, and more than any step.
struct Place {
    uint32_t slot, turn;
    __device__ __forceinline__ Place(uint32_t before, uint32_t c, uint32_t slots) {
        slot = before % slots + c;
        turn = before / slots;
        next(0, slots);
    }
    __device__ __forceinline__ void next(uint32_t step, uint32_t slots) {
        slot += step;
        if (slot >= slots) slot -= slots, ++turn;
    }
    // A wait for a turn by its parity passes wrongly where the turn before has not come yet.  A place therefore has a barrier
    // for even and one for odd turns, and nobody is two turns of the ring ahead of the last chunk that has arrived.
    __device__ __forceinline__ uint64_t* full(uint64_t (*bars)[kMaxSlots]) const { return &bars[turn & 1][slot]; }
    __device__ __forceinline__ uint32_t full_parity() const { return turn >> 1 & 1; }
};

// Two numbers to a block of the cluster, counted by its barrier (which makes them visible to those that wait for it: no
// fence of this block's other writes, which cost 2 us a row)
__device__ __forceinline__ void send_to_block(float* smem, uint64_t* bar, uint32_t rank, float a, float b) {
    uint32_t to, at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(smem)), "r"(rank));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(bar)), "r"(rank));
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(to), "f"(a), "f"(b), "r"(at) : "memory");
}

// A place's barrier is either waiting for a copy, which lands within microseconds, or for none; a wait for both parities,
// each at most about a second, has seen the copy land.
__device__ __forceinline__ void mbar_wait_bounded_short(uint64_t* bar, uint32_t parity) { knn::mbar_wait_bounded(bar, parity, 1u << 18); }

template <class T, bool GIVEN, int kWarps>
__global__ void __launch_bounds__(ring_threads(kWarps), ring_blocks(kWarps)) distill_ring_kernel(Args a) {
    constexpr int kSumWarps = kWarps, kWriteWarps = kWarps;
    extern __shared__ __align__(128) unsigned char ring_smem[];
    __shared__ __align__(8) uint64_t full_bar[2][kMaxSlots], empty_bar[kMaxSlots], stat_bar[kStats], list_bar[kAhead], row_bar[kAhead], free_bar[kAhead];
    __shared__ __align__(8) float stat[GIVEN ? 1 : kStats][(kWarps == 12 ? kMaxRing : 1) * (kSumWarps + 1)][2];  // of warps, then of edges
    __shared__ Factors factors[kAhead];
    __shared__ float4 list_sums[kAhead];
    __shared__ float list_weight[kAhead], list_edge[kAhead][16];
    __shared__ uint32_t list_many[kAhead];
    __shared__ int abort_flag;
    constexpr int E = Row<T>::E;
    const uint32_t size = GIVEN ? 1 : cluster_size(), rank = GIVEN ? 0 : cluster_rank();
    const int lane = threadIdx.x & 31, warp = __shfl_sync(kFull, int(threadIdx.x >> 5), 0);
    const uint64_t items = a.n * (GIVEN ? a.pieces : 1), stride = gridDim.x / size, item0 = blockIdx.x / size;
    constexpr uint32_t kWriters = GIVEN ? kSumWarps + kWriteWarps : kWriteWarps;
    volatile int* aborted = &abort_flag;
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < a.slots; ++s) {
            knn::mbar_init(&full_bar[0][s], 1);
            knn::mbar_init(&full_bar[1][s], 1);
            knn::mbar_init(&empty_bar[s], 1);
        }
        for (int s = 0; s < kAhead; ++s) {
            knn::mbar_init(&list_bar[s], 1);
            knn::mbar_init(&row_bar[s], 1);
            knn::mbar_init(&free_bar[s], kWriters + 1);
        }
        for (int s = 0; s < kStats; ++s) knn::mbar_init(&stat_bar[s], 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (size > 1) {
        cluster_arrive();
        cluster_wait();
    }
    // A block's share of an item: words [w0, w1) of the row.  The warps that sum and write see whole words only; the few
    // logits of a partial word at either end of a row (its edges) are the list's warp's and the row's warp's.
    struct Share {
        Row<T> z;
        uint64_t row;
        uint32_t w0, w1, first, last;  // first, last: words of the row that are whole
        __device__ __forceinline__ Share(const Args& a, uint64_t item, uint32_t rank) : z(a.z, GIVEN ? item / a.pieces : item, a.z_stride, a.rows) {
            row = GIVEN ? item / a.pieces : item;
            const uint32_t piece = GIVEN ? uint32_t(item % a.pieces) : rank;
            w0 = min(z.words, piece * a.per);
            w1 = min(z.words, w0 + a.per);
            first = (z.head + E - 1) / E;
            last = (uint64_t(z.head) + a.rows) % E ? z.words - 1 : z.words;
        }
        __device__ __forceinline__ uint32_t chunks() const { return (w1 - w0 + kChunkWords - 1) / kChunkWords; }
        __device__ __forceinline__ uint32_t from(uint32_t c) const { return max(w0 + c * kChunkWords, first); }
        __device__ __forceinline__ uint32_t to(uint32_t c) const { return max(from(c), min(min(w0 + (c + 1) * kChunkWords, w1), last)); }
        __device__ __forceinline__ int64_t col(uint32_t w) const { return int64_t(w) * E - z.head; }
        // a lane's words of chunk c
        __device__ __forceinline__ void words(uint4 (&x)[8], uint32_t c, const uint4* slot, int lane) const {
            const uint32_t v = w0 + c * kChunkWords + lane, lo = from(c), hi = to(c);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = slot[lane + j * 32];  // (in the ring in any case, whatever it holds)
            if (hi - lo != kChunkWords) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (v + j * 32 < lo || v + j * 32 >= hi) x[j] = nothing<T>();
            }
        }
        __device__ __forceinline__ bool edges() const { return col(first) != 0 || last != z.words; }  // (of the row: the same for all blocks)
        // the column of the edge that is a lane's, or -1
        __device__ __forceinline__ int64_t edge(int lane, uint32_t rows) const {
            if (w0 == w1) return -1;
            const int64_t head_end = w0 == 0 ? col(first) : 0, tail = w1 == z.words ? col(last) + lane - 8 : int64_t(rows);
            return lane < 8 ? (lane < head_end ? lane : -1) : lane < 16 && tail < int64_t(rows) ? tail : -1;
        }
    };
    const uint4* ring = reinterpret_cast<const uint4*>(ring_smem);
    unsigned char* lists = ring_smem + size_t(a.slots) * kChunkBytes;
    uint32_t q = 0;  // chunks of the rows before
    int i = 0;
    bool ok = true;

    if (warp == kSumWarps + kWriteWarps) {
        // (by one thread, a chunk took 400 ns to ask for, half of what the memory needs to bring it)
        if (lane < kCopiers) {
            for (uint64_t item = item0; item < items && ok; item += stride) {
                const Share s(a, item, rank);
                const uint32_t chunks = s.chunks();
                Place at(q, lane, a.slots);
                for (uint32_t c0 = 0; c0 < chunks; c0 += kCopiers, at.next(kCopiers, a.slots)) {
                    const uint32_t c = c0 + lane;
                    if (c < chunks && ok) {
                        ok = mma::wait_or_abort(&empty_bar[at.slot], (at.turn & 1) ^ 1, knn::kWaitLimit, aborted);
                        if (ok) {
                            const uint32_t from = s.from(c), to = s.to(c);
                            const uint32_t bytes = (to - from) * 16;
                            uint64_t* bar = at.full(full_bar);
                            knn::mbar_expect_tx(bar, bytes);
                            if (bytes)
                                knn::bulk_g2s(ring_smem + size_t(at.slot) * kChunkBytes + (from - s.w0 - c * kChunkWords) * 16,
                                              s.z.p + s.col(from), bytes, bar);
                        }
                    }
                    // (in step: none asks for a place's next turn before this one has been asked for)
                    if (__any_sync((1u << kCopiers) - 1, !ok)) {
                        ok = false;
                        break;
                    }
                }
                q += chunks;
            }
        }
    } else if (warp == kSumWarps + kWriteWarps + 1) {
        asm volatile("griddepcontrol.wait;" ::: "memory");  // (the lists' kernel has ended; the others need nothing from it)
        for (uint64_t item = item0; item < items && ok; item += stride, ++i) {
            const int side = i % kAhead;
            // (the writers of a row go ahead of others only as far as its list)
            if (i >= a.ahead) ok = __all_sync(kFull, mma::wait_or_abort(&free_bar[(i - a.ahead) % kAhead], (i - a.ahead) / kAhead & 1, knn::kWaitLimit, aborted));
            if (!ok) break;
            // the list's places in this block's share, from what distill_list_kernel has left
            const Share s(a, item, rank);
            const int64_t from_col = s.col(s.w0), to_col = s.col(s.w1);  // (ids are kept as distances from the first)
            float edge_z = -INFINITY;
            if (s.edges()) {
                const int64_t edge = s.edge(lane, a.rows);
                if (edge >= 0) edge_z = to_float(s.z.p[edge]);
            }
            const List from(a.lists + s.row * list_bytes(a.top), a.top), to(lists + size_t(side) * list_bytes(a.top), a.top);
            const float4 v = a.sums[s.row];
            const float weight = a.weight ? __ldg(a.weight + s.row) : 1.0f;
            uint32_t many = 0;
#pragma unroll 2
            for (uint32_t j0 = 0; j0 < a.top; j0 += 32) {
                const uint32_t j = j0 + lane;
                const bool there = j < a.top;
                const uint32_t id = there ? from.id[j] : kFull;
                const float p = there ? from.p[j] : 0.0f, zj = there ? from.z[j] : 0.0f;
                const bool keep = id != kFull && int64_t(id) >= from_col && int64_t(id) < to_col;
                const uint32_t kept = __ballot_sync(kFull, keep);
                if (keep) {
                    const uint32_t at = many + __popc(kept & ((1u << lane) - 1));
                    to.id[at] = uint32_t(int64_t(id) - from_col);
                    to.p[at] = p;
                    to.z[at] = zj;
                }
                many += __popc(kept);
            }
            if (s.edges()) {
                if (lane < 16) list_edge[side][lane] = edge_z;
                if (!GIVEN) {
                    const float top = warp_max(edge_z), sum = warp_sum(exp2((edge_z - shift_of(top)) * a.c));
                    if (lane < int(size)) send_to_block(stat[i % kStats][size * kSumWarps + rank], &stat_bar[i % kStats], lane, top, sum);
                }
            }
            __syncwarp();
            if (lane == 0) {
                list_sums[side] = v;
                list_weight[side] = weight;
                list_many[side] = many;
                mma::mbar_arrive(&list_bar[side]);
            }
        }
    } else if (warp == kSumWarps + kWriteWarps + 2) {
        for (uint64_t item = item0; item < items && ok; item += stride, ++i) {
            const int side = i % kAhead;
            const Share s(a, item, rank);
            const uint32_t parts_of_row = size * (kSumWarps + (s.edges() ? 1 : 0));
            if (!GIVEN && lane == 0) knn::mbar_expect_tx(&stat_bar[i % kStats], parts_of_row * 8);
            ok = __all_sync(kFull, mma::wait_or_abort(&list_bar[side], i / kAhead & 1, knn::kWaitLimit, aborted));
            if (!ok) break;
            const float4 v = list_sums[side];
            const float weight = list_weight[side];
            MaxSum r;
            if (GIVEN) {
                const float2 st = a.stats[item / a.pieces];
                r.m = st.x;
                r.s = st.y;
            } else {
                ok = __all_sync(kFull, mma::wait_or_abort(&stat_bar[i % kStats], i / kStats & 1, knn::kWaitLimit, aborted));
                if (!ok) break;
                const float(*parts)[2] = stat[i % kStats];
                for (uint32_t b = lane; b < parts_of_row; b += 32) r.m = fmaxf(r.m, parts[b][0]);
                r.m = warp_max(r.m);
                for (uint32_t b = lane; b < parts_of_row; b += 32) r.s += moved(parts[b][1], parts[b][0], r.m, a.c);
                r.s = warp_sum(r.s);
            }
            const Factors f(a.T, weight, r, v.z != 0.0f);
            __syncwarp();
            if (lane == 0) {
                factors[side] = f;
                mma::mbar_arrive(&row_bar[side]);
                if (!GIVEN && rank == 0) a.loss[item] = loss_of(a, ListSums{v.x, v.y, v.z, v.w}, r);
            }
            // the edges' gradients (nobody needs the row's edges any more)
            if (s.edges()) {
                const int64_t edge = s.edge(lane, a.rows);
                T* out = static_cast<T*>(a.grad) + s.row * a.grad_stride;
                if (edge >= 0) out[edge] = from_float<T>(f.zero ? 0.0f : exp2((list_edge[side][lane] - f.shift) * a.c) * f.factor);
                __syncwarp();
                const List list(lists + size_t(side) * list_bytes(a.top), a.top);
                const uint32_t many = f.zero ? 0 : list_many[side];
                for (uint32_t j = lane; j < many; j += 32) {
                    const int64_t id = s.col(s.w0) + list.id[j];
                    if (id < s.col(s.first) || id >= s.col(s.last)) out[id] = from_float<T>(exp2((list.z[j] - f.shift) * a.c) * f.factor - f.taken * list.p[j]);
                }
            }
            __syncwarp();
            if (lane == 0) mma::mbar_arrive(&free_bar[side]);
        }
    } else if (!GIVEN && warp < kSumWarps) {
        for (uint64_t item = item0; item < items && ok; item += stride, ++i) {
            const Share s(a, item, rank);
            const uint32_t chunks = s.chunks();
            if (i >= a.ahead) ok = __all_sync(kFull, mma::wait_or_abort(&free_bar[(i - a.ahead) % kAhead], (i - a.ahead) / kAhead & 1, knn::kWaitLimit, aborted));
            MaxSum acc;
            const uint32_t c0 = (warp + kSumWarps - q % kSumWarps) % kSumWarps;
            Place at(q, c0, a.slots);
            for (uint32_t c = c0; c < chunks && ok; c += kSumWarps, at.next(kSumWarps, a.slots)) {
                ok = __all_sync(kFull, mma::wait_or_abort(at.full(full_bar), at.full_parity(), knn::kWaitLimit, aborted));
                if (!ok) break;
                uint4 x[8];
                s.words(x, c, ring + at.slot * kChunkWords, lane);
                const float top = fmaxf(acc.m, max_of<T>(x));
                acc.s = moved(acc.s, acc.m, top, a.c) + sum_of<T>(x, top, a.c);
                acc.m = top;
            }
            if (!ok) break;
            const float top = warp_max(acc.m);
            const float sum = warp_sum(moved(acc.s, acc.m, top, a.c));
            if (lane < int(size)) send_to_block(stat[i % kStats][rank * kSumWarps + warp], &stat_bar[i % kStats], lane, top, sum);
            q += chunks;
        }
    } else {
        const uint32_t me = GIVEN ? warp : warp - kSumWarps;
        for (uint64_t item = item0; item < items && ok; item += stride, ++i) {
            const Share s(a, item, rank);
            const uint32_t chunks = s.chunks();
            const int side = i % kAhead;
            ok = __all_sync(kFull, mma::wait_or_abort(&row_bar[side], i / kAhead & 1, knn::kWaitLimit, aborted));
            if (!ok) break;
            const Factors f = factors[side];
            const uint32_t many = f.zero ? 0 : list_many[side];
            const List list(lists + size_t(side) * list_bytes(a.top), a.top);
            T* out = static_cast<T*>(a.grad) + s.row * a.grad_stride + s.col(s.w0);  // of the share's first word
            const uint32_t c0 = (me + kWriters - q % kWriters) % kWriters;
            Place at(q, c0, a.slots);
            for (uint32_t c = c0; c < chunks; c += kWriters, at.next(kWriters, a.slots)) {
                ok = __all_sync(kFull, mma::wait_or_abort(at.full(full_bar), at.full_parity(), knn::kWaitLimit, aborted));
                if (!ok) break;
                uint4 x[8];
                s.words(x, c, ring + at.slot * kChunkWords, lane);
                __syncwarp();
                if (lane == 0) mma::mbar_arrive(&empty_bar[at.slot]);
                const uint32_t w = s.w0 + c * kChunkWords + lane, lo = s.from(c), hi = s.to(c);
                T* dst = out + (w - s.w0) * E;
                if (a.same_phase && hi - lo == kChunkWords) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) __stcs(reinterpret_cast<uint4*>(dst + size_t(j) * 32 * E), gradient_of<T>(x[j], f, a.c));
                } else if (a.same_phase) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (w + j * 32 >= lo && w + j * 32 < hi) __stcs(reinterpret_cast<uint4*>(dst + size_t(j) * 32 * E), gradient_of<T>(x[j], f, a.c));
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (w + j * 32 >= lo && w + j * 32 < hi) store_apart<T>(dst + size_t(j) * 32 * E, gradient_of<T>(x[j], f, a.c));
                }
                // the list's ids in this chunk, behind the words that hold them
                const uint32_t lo_off = (lo - s.w0) * E, span = (hi - lo) * E;
                __syncwarp();
                for (uint32_t j = lane; j < many; j += 32) {
                    const uint32_t off = list.id[j];
                    if (off - lo_off < span) out[off] = from_float<T>(exp2((list.z[j] - f.shift) * a.c) * f.factor - f.taken * list.p[j]);
                }
            }
            if (!ok) break;
            __syncwarp();
            if (lane == 0) mma::mbar_arrive(&free_bar[side]);
            q += chunks;
        }
    }
    if (!ok) *aborted = 1;
    __syncwarp();
    __syncthreads();
    if (*aborted && threadIdx.x == 0) atomicExch(a.status, kStatusWaitTimeout);
    // (copies in flight after a lost wait end before the block's memory goes away: that of a place's last turn, or the one before)
    if (*aborted && threadIdx.x < a.slots)
        for (uint32_t k = 0; k < 4; ++k) mbar_wait_bounded_short(&full_bar[k & 1][threadIdx.x], k >> 1);
    __syncthreads();
    if (size > 1) {  // (a block's memory stays until no other can write to it)
        cluster_arrive();
        cluster_wait();
    }
}

// beside: it may begin while the kernel in front of it runs, and waits for that by itself where it has to
template <class K>
int launch_clusters(K* kernel, int threads, const Args& a, uint64_t blocks, uint32_t cluster, uint32_t smem, cudaStream_t st, bool beside = false) {
    CPB_CUDA(allow_max_dynamic_smem(kernel));
    if (cluster > 8) CPB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(blocks));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = beside ? 2 : 1;
    CPB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
    return 0;
}

constexpr uint32_t kRingBytes = 212 * 1024;          // of a block's shared memory, lists included
constexpr uint64_t kPieceWords = 16 * kChunkWords;   // of a row longer than a cluster holds

// Threads for a row: a power of two from 128 to 4,096, as long as all rows' threads run at once (1,024 an SM) and each finds
// words to take.  What one block of up to 512 takes at one go is one block's; else a cluster's blocks are as small as they can
// be, since a block's barriers and its list hold up all of it.  Microseconds with blocks of 128, 256 and 512 threads and the
// best size of cluster for each, bf16: 8,192 rows of 131,072 logits 330, 339, 389 (the memory needs 328), of 20,000 80, 115,
// 158; 1,000 of 100,000 41, 44, 53; 200 of 500,000 43, 45, 48; 16 of 200,000 9.7, 7.9, 7.1; 64 of 32,768 6.2, 6.6, 5.7.
template <class T>
int launch_loss(const Args& a, uint64_t words, cudaStream_t st) {
    int sms = 0;
    CPB_TRY(op::sm_count(&sms));
    uint32_t threads = 128;
    while (threads < 512 * kMaxCluster && a.n * threads * 2 <= uint64_t(sms) * 1024 && uint64_t(threads) * kWords < words) threads *= 2;
    const uint32_t cluster = words <= 512 * kWords ? 1 : threads / 128 < kMaxCluster ? threads / 128 : kMaxCluster;
    const uint32_t bytes = list_bytes(a.top);
    switch (threads / cluster) {
        case 128: return launch_clusters(distill_loss_kernel<T, 128>, 128, a, a.n * cluster, cluster, bytes, st);
        case 256: return launch_clusters(distill_loss_kernel<T, 256>, 256, a, a.n * cluster, cluster, bytes, st);
        default: return launch_clusters(distill_loss_kernel<T, 512>, 512, a, a.n * cluster, cluster, bytes, st);
    }
}
template <class T, int kHeld>
int launch_short(const Args& a, uint32_t smem, cudaStream_t st) {
    auto kernel = distill_short_kernel<T, kHeld>;
    CPB_CUDA(allow_max_dynamic_smem(kernel));
    kernel<<<unsigned((a.n + kShortWarps - 1) / kShortWarps), kShortWarps * 32, smem, st>>>(a);
    CPB_CUDA(cudaGetLastError());
    return 0;
}
// shared memory of a block, at most: what lists leave goes to the ring
constexpr uint32_t ring_bytes(int warps) { return kRingBytes / ring_blocks(warps) - (ring_blocks(warps) - 1) * 4096; }
// places of a ring, beside the lists
template <int kWarps>
uint32_t ring_slots(uint32_t top) {
    const uint32_t bytes = ring_bytes(kWarps), lists = kAhead * list_bytes(top);
    const uint32_t slots = bytes > lists ? (bytes - lists) / kChunkBytes : 0;
    return slots < kMaxSlots ? slots : kMaxSlots;
}
// Words of a row that a block may have: as many chunks as, together with the next row's, the ring holds when every writer has
// taken one of the first.  (With two chunks more the next row's last copies wait for the writers' second turn: 131,072 bf16
// logits in halves of 32 chunks, 8,192 rows: ring of 52 chunks 675 us, of 50 chunks 880 us.)
template <int kWarps>
uint64_t ring_share(uint32_t top) {
    const uint32_t slots = ring_slots<kWarps>(top);
    return slots <= kWarps ? 0 : uint64_t(slots + kWarps) / 2 * kChunkWords;
}
// Clusters of the ring's kernel that run at once, asked for once per device and size of cluster.  The length of the lists does not
// come into it: a ring takes what they leave but for less than a place, or 52 places, so that an SM has room for ring_blocks blocks
// and no more whatever the length.  (Asked for again with every length, eleven sizes took the host 4.7 us of 21 a call.)
template <class T, bool GIVEN, int kWarps>
int clusters_at_once(uint32_t cluster, uint64_t* out) {
    static_assert(ring_blocks(kWarps) * ring_bytes(kWarps) < 227 * 1024 && (ring_blocks(kWarps) + 1) * (ring_bytes(kWarps) - kChunkBytes) > 227 * 1024 &&
                      (ring_bytes(kWarps) < kMaxSlots * kChunkBytes || (ring_blocks(kWarps) + 1) * kMaxSlots * kChunkBytes > 227 * 1024),
                  "blocks an SM");
    static std::atomic<int> known[op::kMaxDevices][kMaxRing + 1];
    int dev = 0;
    CPB_CUDA(cudaGetDevice(&dev));
    int many = known[dev][cluster].load(std::memory_order_relaxed);
    if (!many) {
        auto kernel = distill_ring_kernel<T, GIVEN, kWarps>;
        CPB_CUDA(allow_max_dynamic_smem(kernel));
        if (cluster > 8) CPB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(cluster);
        cfg.blockDim = dim3(ring_threads(kWarps));
        cfg.dynamicSmemBytes = ring_bytes(kWarps);
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = cluster;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        CPB_CUDA(cudaOccupancyMaxActiveClusters(&many, kernel, &cfg));
        if (many < 1) many = 1;
        known[dev][cluster].store(many, std::memory_order_relaxed);
    }
    *out = many;
    return 0;
}
template <class T, bool GIVEN, int kWarps>
int launch_ring(Args& a, uint64_t words, uint32_t parts, cudaStream_t st) {
    a.slots = ring_slots<kWarps>(a.top);
    const uint32_t smem = a.slots * kChunkBytes + kAhead * list_bytes(a.top);
    auto kernel = distill_ring_kernel<T, GIVEN, kWarps>;
    uint64_t most = 0;
    if (GIVEN) {
        CPB_TRY((clusters_at_once<T, GIVEN, kWarps>(1, &most)));
    } else {
        // More blocks a row than it takes, where clusters of that size leave SMs over that larger ones do not (their SMs have to
        // lie together): 1,000 rows of 700,001 bf16 logits, 11 blocks a row 784 us, 16 549.  3, 5, 6 and 7 are left out: as many
        // clusters as are counted for them do not run at once, and the last ones' rows come when the others' are done (2,000 rows
        // of 180,000: by threes 452 us, by fours 240; 1,000 of 300,000: by fives or sixes 384 us, by nines 210).
        uint64_t used = 0;
        uint32_t best = parts;
        for (uint32_t size = parts; size <= (parts == 1 ? 1 : kMaxRing); ++size) {
            if (size < 8 && (size & (size - 1)) != 0) continue;
            uint64_t many = 0;
            CPB_TRY((clusters_at_once<T, GIVEN, kWarps>(size, &many)));
            if (many * size * 32 > used * 33) used = many * size, best = size, most = many;
        }
        parts = best;
    }
    a.per = (uint32_t((words + parts - 1) / parts) + 7) / 8 * 8;  // (shares start on lines)
    a.pieces = parts;
    const uint32_t chunks = (a.per + kChunkWords - 1) / kChunkWords, ahead = 2 * a.slots / chunks;  // (two turns of the ring; see Place)
    a.ahead = int(ahead < kAhead ? ahead : kAhead);
    CPB_TRY(op::status_word(&a.status));
    const uint32_t cluster = GIVEN ? 1 : parts;
    const uint64_t items = GIVEN ? a.n * parts : a.n;
    return launch_clusters(kernel, ring_threads(kWarps), a, (items < most ? items : most) * cluster, cluster, smem, st, !GIVEN);
}

template <class T>
int launch_distill(Args& a, cudaStream_t st) {
    constexpr uint32_t E = 16 / sizeof(T);
    // 16-byte words of a row, from the start of its first 128-byte line on
    const bool aligned = op::Alignment().add(a.z).add(a.n > 1 ? a.z_stride * sizeof(T) : uint64_t(0)).holds(128);
    const uint64_t words = (uint64_t(a.rows) + (aligned ? 0 : 8 * E - 1) + E - 1) / E;
    CPB_OP_CHECK(a.n * kMaxRing < (1ull << 31), "distill: too many rows for one call");
    const uint32_t list_smem = kListWarps * (list_bytes(a.top) + table_words(a.top) * 4);
    static_assert(kListWarps == kShortWarps, "one size of shared memory for both");
    const unsigned list_blocks = unsigned((a.n + kListWarps - 1) / kListWarps);
    // (4,000 bf16 logits, 8,192 rows: 47 us in registers, 14 + 52 by lists and a ring; 5,000 logits do not fit)
    // (the loss alone by a warp a row, and by a block of 128: 8,192 rows of 1,000 bf16 logits 11 us and 39, of 4,000 24 and 41; 148
    // rows 4.1 and 5.2, 5.4 and 5.3)
    if (!a.grad && words > 32 * 16) return launch_loss<T>(a, words, st);
    if (words <= 32 * 3) return launch_short<T, 3>(a, list_smem, st);
    if (words <= 32 * 6) return launch_short<T, 6>(a, list_smem, st);
    if (words <= 32 * 10) return launch_short<T, 10>(a, list_smem, st);
    if (words <= 32 * 16) return launch_short<T, 16>(a, list_smem, st);
    CPB_CUDA(allow_max_dynamic_smem(distill_list_kernel<T>));
    distill_list_kernel<T><<<list_blocks, kListWarps * 32, list_smem, st>>>(a);
    CPB_CUDA(cudaGetLastError());
    // Three small blocks an SM for rows of up to five chunks, 8,192 rows of bf16 each: 5,000 logits 63 us (one large block 131),
    // 8,192 logits 70 (98); 16,384 logits 116 (104).
    if (words <= 5 * kChunkWords && words <= ring_share<3>(a.top)) return launch_ring<T, false, 3>(a, words, 1, st);
    const uint64_t share = ring_share<12>(a.top), parts = (words + share - 1) / share;
    if (parts <= kMaxRing) return launch_ring<T, false, 12>(a, words, uint32_t(parts), st);
    CPB_TRY(launch_loss<T>(a, words, st));
    const uint64_t pieces = (words + kPieceWords - 1) / kPieceWords;
    CPB_OP_CHECK(a.n * pieces < (1ull << 31), "distill: too many rows for one call");
    return launch_ring<T, true, 12>(a, words, uint32_t(pieces), st);
}

int distill(const char* what, Args& a, const void* d_logits, int type, uint64_t n, uint64_t rows, uint64_t stride, const void* d_ids,
            uint32_t id_bytes, uint64_t ids_stride, const float* d_teacher, uint64_t teacher_stride, uint64_t top, float temperature,
            float* d_loss, cudaStream_t st) {
    char text[160];
    auto bad = [&](const char* why) {
        snprintf(text, sizeof text, "%s: %s", what, why);
        return op::invalid(text);
    };
    if (!op::type_known(type)) return bad("unknown element type");
    if (id_bytes != 4 && id_bytes != 8) return bad("ids have 4 or 8 bytes");
    if (rows < 1 || rows >= (1ull << 31)) return bad("need 1 <= rows < 2^31");
    if (top > kMaxTop) return bad("a list has at most 1,024 places");
    if (!(temperature > 0.0f) || !(temperature < INFINITY)) return bad("the temperature must be positive and finite");
    if (n == 0) return 0;
    if (n >= (1ull << 31)) return bad("too many rows for one call");
    if (!d_logits || !d_loss || (top && (!d_ids || !d_teacher))) return bad("null pointer");
    if (!op::Alignment().add(d_logits).add(a.grad).holds(op::type_bytes(type)) || !op::Alignment().add(d_teacher).add(d_loss).add(a.weight).holds(4) ||
        !op::Alignment().add(d_ids).holds(id_bytes))
        return bad("an address is no multiple of its element's size");
    CPB_TRY(op::check_device());
    a.z = d_logits;
    a.ids = {d_ids, id_bytes, uint32_t(rows)};
    a.teacher = d_teacher;
    a.loss = d_loss;
    a.n = n;
    a.z_stride = stride;
    a.ids_stride = ids_stride;
    a.teacher_stride = teacher_stride;
    a.rows = uint32_t(rows);
    a.top = uint32_t(top);
    a.T = temperature;
    a.c = kLog2e / temperature;
    a.same_phase = op::Alignment().add(uint64_t(reinterpret_cast<uintptr_t>(d_logits) - reinterpret_cast<uintptr_t>(a.grad))).add((stride - a.grad_stride) * op::type_bytes(type)).holds(16);
    switch (type) {
        case CPHNSW_B200_F32: return launch_distill<float>(a, st);
        case CPHNSW_B200_F16: return launch_distill<__half>(a, st);
        default: return launch_distill<__nv_bfloat16>(a, st);
    }
}

}  // namespace
}  // namespace cpb

using namespace cpb;

extern "C" {

int cphnsw_b200_distill_loss_dev(const void* d_logits, int type, uint64_t n, uint64_t rows, uint64_t logits_stride,
                                 const void* d_ids, uint32_t id_bytes, uint64_t ids_stride, const float* d_teacher,
                                 uint64_t teacher_stride, uint64_t top, float temperature, float* d_loss, void* stream) {
    Args a{};
    return distill("distill_loss", a, d_logits, type, n, rows, logits_stride, d_ids, id_bytes, ids_stride, d_teacher, teacher_stride,
                   top, temperature, d_loss, static_cast<cudaStream_t>(stream));
}

uint64_t cphnsw_b200_distill_workspace(uint64_t n, uint64_t top) { return n * (sizeof(float4) + sizeof(float2) + list_bytes(uint32_t(top))); }

int cphnsw_b200_distill_loss_and_grad_dev(const void* d_logits, int type, uint64_t n, uint64_t rows, uint64_t logits_stride,
                                          const void* d_ids, uint32_t id_bytes, uint64_t ids_stride, const float* d_teacher,
                                          uint64_t teacher_stride, uint64_t top, float temperature, const float* d_weight,
                                          float* d_loss, void* d_grad, uint64_t grad_stride, void* d_workspace,
                                          uint64_t workspace_bytes, void* stream) {
    Args a{};
    CPB_OP_CHECK(d_grad || n == 0, "distill_loss_and_grad: null pointer");
    CPB_OP_CHECK(grad_stride >= rows || n <= 1, "distill_loss_and_grad: rows of the gradient overlap");
    if (n < (1ull << 31) && top <= kMaxTop) {  // (else refused below)
        const uint64_t need = cphnsw_b200_distill_workspace(n, top);
        CPB_OP_CHECK(workspace_bytes >= need && (need == 0 || (d_workspace && op::Alignment().add(d_workspace).holds(16))),
                     "distill_loss_and_grad: the workspace is too small, or not aligned to 16 bytes");
    }
    a.grad = d_grad;
    a.grad_stride = grad_stride;
    a.weight = d_weight;
    a.sums = static_cast<float4*>(d_workspace);
    a.stats = reinterpret_cast<float2*>(a.sums + n);
    a.lists = reinterpret_cast<unsigned char*>(a.stats + n);
    return distill("distill_loss_and_grad", a, d_logits, type, n, rows, logits_stride, d_ids, id_bytes, ids_stride, d_teacher,
                   teacher_stride, top, temperature, d_loss, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
