// Distillation from a teacher's best k: Kullback-Leibler loss of rows of logits, and its gradient.
//
// A row's teacher is a list of k (column, score) pairs -- what an exact search leaves in device memory --
// with p = softmax(t / T) over the list; the student is q = softmax(z / T) over all columns.
//
//   loss = T^2 sum_j p_j (log p_j - log q_{id_j}),      d loss / d z_c = T (q_c - sum_{j: id_j = c} p_j).
//
// The loss needs two numbers of the whole row, m = max z and ln sum exp((z - m) / T), and k logits; the
// gradient needs the row again. Bound by HBM: one read of the logits for the loss, one read and one write
// for a gradient. Rows of up to 65536 columns stay in registers between the sum and the gradient; longer rows
// are cut into chunks, each in the registers of one workgroup, whose partial (m, sum) pairs are joined by a second
// launch, the gradient's where there is one, which reads the logits again; a gradient over more than 1024 chunks a row
// takes three (parts, joining, gradient).
//
// Exponentials go through exp2 of (z - m) log2(e) / T: the difference first, so that rows at the type's lowest
// value, whose product with 1 / T would overflow, still come out as the distribution they are. Sums over a
// row are 32-bit per thread, 64-bit across threads, and a chunk's is rounded to 32 bits once more where it goes to memory: 24 or
// 34 roundings of 2^-24 a row, beside the exponentials' own. The teacher's exponentials are 32-bit (3 * 2^-24, the hardware's
// exp2), their sums, over a repeated id too, and the differences of logits they weight 64-bit.
#include <algorithm>
#include "trag_ops.h"

namespace trag {
namespace {

// f32 here goes by eight elements too, two 16-byte accesses a vector: half the branches of a row (4096 x 32000, loss and
// gradient: 207 us, by four 239)
struct F32by8 {
    typedef float elem;
    static constexpr int W = 8;
    typedef float vec __attribute__((ext_vector_type(8), aligned(4)));
    static __device__ __forceinline__ float round(float v) { return v; }
};

constexpr uint32_t LIST_MAX = 1024;        // teacher entries per row
constexpr uint32_t ROW_MAX = 65536;        // columns of the row kernel
constexpr uint32_t PART_STEP = 2048;       // a chunk of a long row is a multiple of this
// ... and at most what 256 threads hold as four vectors each (gradient of 4096 x 32000 bf16: 102 us, 5.1 TB/s; two vectors
// 125, eight 102; reading the logits where each is needed 116)
constexpr int PART_VECS = 4;
constexpr uint32_t JOIN_MAX = 1024u;       // chunks of a row whose parts the gradient's workgroups join themselves
constexpr uint32_t PART_MAX = 256u * 8u * PART_VECS;

struct DistillArgs {
    const void* z;
    const uint32_t* ids;
    const float* teacher;
    const uint32_t* counts;
    float* loss;
    float* norm;              // 2 per row: max, ln sum exp((z - max) / T)
    const float* norm_in;     // the same, for the gradient alone
    const float* weight;      // per row, null: 1
    void* grad;
    float* parts;             // 2 per row and chunk, behind them 4 per row (list_part)
    uint64_t z_stride, grad_stride;
    uint32_t n_rows, n_cols, k, chunk, n_chunks;
    uint32_t row0;            // first row of a launch
    uint32_t slot_mask;       // slots of the id table, a power of two, less one
    float temperature, c;     // c = log2(e) / T
    double c64;
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// exponent of e^((z - m) / T) as a power of two (off by three roundings, 3 * 2^-24 relative; an infinite z stays what it is)
__device__ __forceinline__ float expo(const DistillArgs& a, float z, float m) { return (z - m) * a.c; }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// 2^x of a list's entry, to 3 * 2^-24: the whole part of x goes to the exponent, what is left is below one half
__device__ __forceinline__ float list_exp(double x) {
    if (x < -126.0) return 0.0f;
    const double n = __builtin_rint(x);
    return __builtin_ldexpf(exp2_hw((float)(x - n)), (int)n);
}

// Where a workgroup's waves meet: maxima of the row and of its teacher list, then three sums.
template <int NW>
struct Meet {
    float top[2][NW];
    double sum[3][NW];
};

// A row's teacher list in LDS, which is sized by the call: ids (NO_ID: an entry behind the row's count, or no column),
// scores and later their exponentials, the logits at the ids. Entry j belongs to thread j % NT throughout. Behind it, for a
// gradient, the first entry of every id and whether the id comes again: an open hash table of at least twice as many
// slots as entries, filled anew for every row. Slots depend on who came first, what they say does not.
struct List {
    uint32_t* id;
    float* e;
    float* z;
    uint32_t* slot_id;
    uint32_t* slot_first;
    uint32_t* slot_again;     // a bit a slot
    __device__ __forceinline__ List(const DistillArgs& a, uint32_t* lds)
        : id(lds), e(reinterpret_cast<float*>(lds + a.k)), z(reinterpret_cast<float*>(lds + 2u * a.k)), slot_id(lds + 3u * a.k),
          slot_first(slot_id + a.slot_mask + 1u), slot_again(slot_first + a.slot_mask + 1u) {}
};
inline uint32_t list_bytes(const DistillArgs& a, bool table) {
    return 4u * (3u * a.k + (table ? 2u * (a.slot_mask + 1u) + (a.slot_mask + 1u) / 32u : 0u));
}
constexpr uint32_t NO_ID = 0xFFFFFFFFu;   // (never a column: columns are below the number of columns)

// p = softmax(t / T) over the list. `some`: the list has probability at all (an empty list, or one of minus
// infinities, leaves the row out: loss and gradient 0).
template <int NT>
struct Teacher {
    uint32_t id0;
    float t0;
    double sum;      // sum e, e = exp((t - max t) / T)
    double cross;    // sum e ((t - max t) / T - (z_id - max z) / T)
    bool some;

    // Asked for ahead of the row: the first NT entries (whatever the row's count, so that the loads need not wait for it).
    __device__ __forceinline__ void ask(const DistillArgs& a, uint64_t row) {
        id0 = NO_ID;
        t0 = 0.0f;
        if (threadIdx.x < a.k) {
            id0 = a.ids[row * a.k + threadIdx.x];
            t0 = a.teacher[row * a.k + threadIdx.x];
        }
        const uint32_t n = a.counts ? min(a.counts[row], a.k) : a.k;
        if (threadIdx.x >= n || id0 >= a.n_cols) id0 = NO_ID;
        this->n = n;
    }
    // The list into LDS, with the logits of the ids in [c0, c1); the largest score of this thread's entries.
    template <typename T>
    __device__ __forceinline__ float take(const DistillArgs& a, uint64_t row, const typename T::elem* z, uint32_t c0, uint32_t c1, const List& l) {
        float top = -INFINITY;
        uint32_t id = id0;
        float t = t0;
        for (uint32_t j = threadIdx.x; j < a.k; j += NT) {
            if (j >= NT) {
                id = a.ids[row * a.k + j];
                t = a.teacher[row * a.k + j];
                if (j >= n || id >= a.n_cols) id = NO_ID;
            }
            l.id[j] = id;
            l.e[j] = t;
            l.z[j] = id != NO_ID && id >= c0 && id < c1 ? (float)z[id] : 0.0f;
            if (id != NO_ID) top = fmaxf(top, t);   // (a NaN passes the maximum by and reaches the loss through its exponential)
        }
        return top;
    }
    // this thread's part of the two sums; the exponentials replace the scores
    __device__ __forceinline__ void sums(const DistillArgs& a, float top, float ref, const List& l) {
        const float s0 = top == -INFINITY ? 0.0f : top;   // (a list of minus infinities: every difference would be NaN)
        sum = cross = 0.0;
        for (uint32_t j = threadIdx.x; j < a.k; j += NT) {
            const float e = l.id[j] != NO_ID ? list_exp(((double)l.e[j] - (double)s0) * a.c64) : 0.0f;
            sum += (double)e;
            // (1 / T comes with the sum: write_row)
            if (!(e == 0.0f)) cross += (double)e * (((double)l.e[j] - (double)s0) - ((double)l.z[j] - (double)ref));
            l.e[j] = e;
        }
    }
    static __device__ __forceinline__ void clear(const DistillArgs& a, const List& l) {
        for (uint32_t s = threadIdx.x; s <= a.slot_mask; s += NT) {
            l.slot_id[s] = NO_ID;
            l.slot_first[s] = NO_ID;
            if ((s & 31u) == 0u) l.slot_again[s >> 5] = 0u;
        }
    }
    static __device__ __forceinline__ uint32_t home(const DistillArgs& a, uint32_t id) { return (id * 2654435761u) >> 21 & a.slot_mask; }
    // (a barrier after clear, and one before patch)
    static __device__ __forceinline__ void enter(const DistillArgs& a, const List& l, uint32_t c0, uint32_t c1) {
        for (uint32_t j = threadIdx.x; j < a.k; j += NT) {
            const uint32_t id = l.id[j];
            if (id == NO_ID || id < c0 || id >= c1) continue;
            uint32_t s = home(a, id), was;
            while ((was = atomicCAS(&l.slot_id[s], NO_ID, id)) != NO_ID && was != id) s = (s + 1u) & a.slot_mask;   // (half of the slots are free)
            if (was == id) atomicOr(&l.slot_again[s >> 5], 1u << (s & 31u));
            atomicMin(&l.slot_first[s], j);
        }
    }
    // (after the sums of all threads are in)
    __device__ __forceinline__ void finish() { some = !(sum == 0.0); }
    // The gradient at the list's columns, after everything else of [c0, c1) has been written: the first entry of an id
    // takes the probabilities of all entries of that id, in the list's order. (The logits there come from the list: the
    // gradient may have gone in their place.)
    template <typename T>
    __device__ __forceinline__ void patch(const DistillArgs& a, const List& l, typename T::elem* g, uint32_t c0, uint32_t c1,
                                          float ref, float per_sum, float gt) const {
        const double inv64 = 1.0 / sum;
        const float inv = (float)inv64;
        for (uint32_t j = threadIdx.x; j < a.k; j += NT) {
            const uint32_t id = l.id[j];
            if (id == NO_ID || id < c0 || id >= c1) continue;
            uint32_t s = home(a, id);
            while (l.slot_id[s] != id) s = (s + 1u) & a.slot_mask;   // (it has been entered)
            if (l.slot_first[s] != j) continue;
            float p = l.e[j] * inv;
            // (up to 1024 terms: in 32 bits they lost up to 25 * 2^-24. Eight entries' loads ahead of their additions: 1000 x 32000
            // bf16, lists of 1024 entries on one column 76 us, entry by entry 124)
            if (l.slot_again[s >> 5] >> (s & 31u) & 1u) {
                double e = (double)l.e[j];
                uint32_t o = j + 1u;
                for (; o + 8u <= a.k; o += 8u) {
                    float v[8];
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) v[i] = l.e[o + i];
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) v[i] = l.id[o + i] == id ? v[i] : 0.0f;
#pragma unroll
                    for (uint32_t i = 0; i < 8u; ++i) e += (double)v[i];
                }
                for (; o < a.k; ++o) e += l.id[o] == id ? (double)l.e[o] : 0.0;
                p = (float)(e * inv64);
            }
            g[id] = T::round(gt * (exp2_hw(expo(a, l.z[j], ref)) * per_sum - p));
        }
    }

  private:
    uint32_t n;
};

// what a row's sums come to: loss = T^2 (sum p (log p - log q)) = T^2 (cross / sum / T - log sum + log of the row's sum)
template <int NT>
__device__ __forceinline__ void write_row(const DistillArgs& a, uint64_t row, float m, double row_sum, const Teacher<NT>& l) {
    const double ln = log(row_sum), temp = (double)a.temperature;
    a.loss[row] = l.some ? (float)(temp * (l.cross / l.sum) + temp * temp * (ln - log(l.sum))) : 0.0f;
    a.norm[2 * row] = m;
    a.norm[2 * row + 1] = (float)ln;
}

// 16-bit types: what is carried on is the row as it is in memory; without this the compiler keeps the converted floats
// from one pass to the next, in twice the registers
template <typename T, int NV>
__device__ __forceinline__ void keep_raw(typename T::vec (&h)[NV]) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    if constexpr (sizeof(typename T::elem) == 2) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            u32x4 w = __builtin_bit_cast(u32x4, h[v]);
            asm volatile("" : "+v"(w));
            h[v] = __builtin_bit_cast(typename T::vec, w);
        }
    }
}

// One workgroup a row, the row in registers as NV vectors of W columns a thread (the columns behind the last
// whole vector: one each for the first few threads): one read of the logits, one write of the gradient, two meetings
// of the waves and one more before the list's columns are set right. (Sixteen 16-bit vectors of eight waves are held to 128
// registers, so that two rows fit a CU: 1000 x 50257 bf16 with the gradient 60 us. Without the bound they take 134, one row a CU, 67
// us; the bound costs six registers, 28 bytes of scratch a thread. With a loop over rows they took 194, 72 us.)
template <typename T, int NT, int NV, bool GRAD>
__global__ void __launch_bounds__(NT, NT == 512 && sizeof(typename T::elem) == 2 ? 4 : 1) distill_row_kernel(const DistillArgs a) {
    typedef typename T::elem E;
    constexpr int NW = NT / 64;
    __shared__ Meet<NW> meet;
    extern __shared__ uint32_t lds[];
    const List list(a, lds);
    const uint32_t wid = threadIdx.x >> 6;
    const bool lead = (threadIdx.x & 63u) == 0u;
    const uint32_t whole = a.n_cols / T::W * T::W, ct = whole + threadIdx.x;
    const uint64_t row = (uint64_t)a.row0 + blockIdx.x;
    const E* const z = reinterpret_cast<const E*>(a.z) + row * a.z_stride;
    Teacher<NT> l;
    l.ask(a, row);
    // (held as they are in memory; in f32 the exponentials take their place, 16-bit types compute them again for the
    // gradient, which costs less than the occupancy that twice the registers would)
    typename T::vec h[NV];
    float et = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const uint32_t c = ((uint32_t)v * NT + threadIdx.x) * T::W;
        h[v] = fill_vec<T>(-INFINITY);
        if (c < whole) h[v] = load_vec<T>(z + c);
    }
    if (threadIdx.x < (uint32_t)T::W && ct < a.n_cols) et = (float)z[ct];
    if constexpr (GRAD) l.clear(a, list);
    float lt = wave_max(l.template take<T>(a, row, z, 0u, a.n_cols, list));
    float m = et;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < T::W; ++i) m = fmaxf(m, (float)h[v][i]);
    keep_raw<T, NV>(h);
    m = wave_max(m);
    if (lead) { meet.top[0][wid] = m; meet.top[1][wid] = lt; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) { m = fmaxf(m, meet.top[0][w]); lt = fmaxf(lt, meet.top[1][w]); }
    const float ref = m == -INFINITY ? 0.0f : m;
    if constexpr (GRAD) l.enter(a, list, 0u, a.n_cols);
    l.sums(a, lt, ref, list);
    et = exp2_hw(expo(a, et, ref));
    float s = et;   // (a vector's sum first: an exponential goes through at most W + NV additions in 32 bits)
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        float sv = 0.0f;
#pragma unroll
        for (int i = 0; i < T::W; ++i) {
            const float x = exp2_hw(expo(a, (float)h[v][i], ref));
            sv += x;
            if constexpr (GRAD && sizeof(E) == 4) h[v][i] = x;
        }
        s += sv;
    }
    if constexpr (GRAD) keep_raw<T, NV>(h);
    double sum = wave_sum((double)s);
    l.sum = wave_sum(l.sum);
    l.cross = wave_sum(l.cross);
    if (lead) { meet.sum[0][wid] = sum; meet.sum[1][wid] = l.sum; meet.sum[2][wid] = l.cross; }
    __syncthreads();
    sum = l.sum = l.cross = 0.0;
#pragma unroll
    for (int w = 0; w < NW; ++w) { sum += meet.sum[0][w]; l.sum += meet.sum[1][w]; l.cross += meet.sum[2][w]; }
    l.finish();
    if constexpr (GRAD) {
        E* const g = reinterpret_cast<E*>(a.grad) + row * a.grad_stride;
        const float gt = a.temperature * (a.weight ? a.weight[row] : 1.0f);
        const float f = (float)((double)gt / sum);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const uint32_t c = ((uint32_t)v * NT + threadIdx.x) * T::W;
            typename T::vec o;
#pragma unroll
            for (int i = 0; i < T::W; ++i) {
                const float x = sizeof(E) == 4 ? (float)h[v][i] : exp2_hw(expo(a, (float)h[v][i], ref));
                o[i] = T::round(l.some ? x * f : 0.0f);
            }
            if (c < whole) store_vec<T>(g + c, o);
        }
        if (threadIdx.x < (uint32_t)T::W && ct < a.n_cols) g[ct] = T::round(l.some ? et * f : 0.0f);
        // what the workgroup has written so far is in memory, in front of what follows
        __threadfence_block();
        __syncthreads();
        if (l.some) l.template patch<T>(a, list, g, 0u, a.n_cols, ref, (float)(1.0 / sum), gt);
    }
    if (threadIdx.x == 0) write_row(a, row, m, sum, l);
}

// What a row's list comes to before the row's maximum is known, behind the parts: a double, the sum of
// e ((t - max t) - (z_id - zl)), and zl, the list's largest logit -- differences of logits, which lose nothing where the logits are huge.
__device__ __forceinline__ float* list_part(const DistillArgs& a, uint64_t row) { return a.parts + 2 * (uint64_t)a.n_rows * a.n_chunks + 4 * row; }

// (max, sum) of one chunk of one row; a chunk is at most PART_VECS vectors a thread. LIST: a row's first chunk does the list's
// part of the loss too, while the logits are what they were (a gradient may go in their place).
template <typename T, int NT, bool LIST>
__global__ void __launch_bounds__(NT) distill_part_kernel(const DistillArgs a) {
    typedef typename T::elem E;
    constexpr int NW = NT / 64;
    __shared__ Meet<NW> meet;
    const uint32_t wid = threadIdx.x >> 6;
    const bool lead = (threadIdx.x & 63u) == 0u;
    const uint64_t part = (uint64_t)a.row0 * a.n_chunks + blockIdx.x, row = part / a.n_chunks;
    const uint64_t c0 = (part % a.n_chunks) * a.chunk;
    extern __shared__ uint32_t lds[];
    const List list(a, lds);
    Teacher<NT> l;
    const bool first = LIST && c0 == 0;   // (of the whole workgroup)
    if (first) l.ask(a, row);
    const uint32_t n = (uint32_t)min((uint64_t)a.chunk, a.n_cols - c0);
    const E* const z = reinterpret_cast<const E*>(a.z) + row * a.z_stride + c0;
    const uint32_t whole = n / T::W * T::W, ct = whole + threadIdx.x;   // (the columns behind the last whole vector, one each)
    typename T::vec h[PART_VECS];
    float et = -INFINITY;
#pragma unroll
    for (int v = 0; v < PART_VECS; ++v) {
        const uint32_t c = ((uint32_t)v * NT + threadIdx.x) * T::W;
        h[v] = fill_vec<T>(-INFINITY);
        if (c < whole) h[v] = load_vec<T>(z + c);
    }
    if (threadIdx.x < (uint32_t)T::W && ct < n) et = (float)z[ct];
    if constexpr (LIST) {
        if (first) {
            float lt = wave_max(l.template take<T>(a, row, z, 0u, a.n_cols, list)), zl = -INFINITY;
            for (uint32_t j = threadIdx.x; j < a.k; j += NT)
                if (list.id[j] != NO_ID) zl = fmaxf(zl, list.z[j]);
            zl = wave_max(zl);
            if (lead) { meet.top[0][wid] = zl; meet.top[1][wid] = lt; }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; ++w) { zl = fmaxf(zl, meet.top[0][w]); lt = fmaxf(lt, meet.top[1][w]); }
            if (zl == -INFINITY) zl = 0.0f;
            l.sums(a, lt, zl, list);
            l.cross = wave_sum(l.cross);
            if (lead) meet.sum[1][wid] = l.cross;
            __syncthreads();
            if (threadIdx.x == 0) {
                l.cross = 0.0;
#pragma unroll
                for (int w = 0; w < NW; ++w) l.cross += meet.sum[1][w];
                float* const to = list_part(a, row);   // (4-byte aligned: the two words of a double)
                const uint64_t bits = __builtin_bit_cast(uint64_t, l.cross);
                to[0] = __builtin_bit_cast(float, (uint32_t)bits);
                to[1] = __builtin_bit_cast(float, (uint32_t)(bits >> 32));
                to[2] = zl;
            }
        }
    }
    float m = et;
#pragma unroll
    for (int v = 0; v < PART_VECS; ++v)
#pragma unroll
        for (int i = 0; i < T::W; ++i) m = fmaxf(m, (float)h[v][i]);
    // (each wave's sum at its own maximum, then the waves' at the workgroup's)
    m = wave_max(m);
    const float ref = m == -INFINITY ? 0.0f : m;
    float s = exp2_hw(expo(a, et, ref));
#pragma unroll
    for (int v = 0; v < PART_VECS; ++v)
#pragma unroll
        for (int i = 0; i < T::W; ++i) s += exp2_hw(expo(a, (float)h[v][i], ref));
    const double ws = wave_sum((double)s);
    if (lead) { meet.top[0][wid] = m; meet.sum[0][wid] = ws; }
    __syncthreads();
    if (threadIdx.x == 0) {
        float top = meet.top[0][0];
#pragma unroll
        for (int w = 1; w < NW; ++w) top = fmaxf(top, meet.top[0][w]);
        double sum = 0.0;
#pragma unroll
        for (int w = 0; w < NW; ++w)   // (a wave without a number: its sum is 0, or NaN, and stays that)
            sum += meet.sum[0][w] * (meet.top[0][w] == -INFINITY ? 1.0 : (double)exp2_hw(expo(a, meet.top[0][w], top)));
        a.parts[2 * part] = top;
        a.parts[2 * part + 1] = (float)sum;   // (one rounding beside the 33 of a thread's own sum; the pair stays 8 bytes)
    }
}

// this thread's part of a row's chunks: their maximum, and their sums brought to the row's maximum
template <int NT>
__device__ __forceinline__ float parts_max(const DistillArgs& a, uint64_t row) {
    const float* const parts = a.parts + 2 * row * a.n_chunks;
    float m = -INFINITY;
    for (uint32_t c = threadIdx.x; c < a.n_chunks; c += NT) m = fmaxf(m, parts[2 * c]);
    return m;
}
template <int NT>
__device__ __forceinline__ double parts_sum(const DistillArgs& a, uint64_t row, float ref) {
    const float* const parts = a.parts + 2 * row * a.n_chunks;
    double sum = 0.0;
    for (uint32_t c = threadIdx.x; c < a.n_chunks; c += NT) {
        const float pm = parts[2 * c];
        // (a chunk without a number: its sum is 0, or NaN, and stays that)
        sum += (double)parts[2 * c + 1] * (pm == -INFINITY ? 1.0 : (double)exp2_hw(expo(a, pm, ref)));
    }
    return sum;
}

// a row's chunks joined, and its loss
template <typename T, int NT>
__global__ void __launch_bounds__(NT) distill_join_kernel(const DistillArgs a) {
    typedef typename T::elem E;
    constexpr int NW = NT / 64;
    __shared__ Meet<NW> meet;
    extern __shared__ uint32_t lds[];
    const List list(a, lds);
    const uint32_t wid = threadIdx.x >> 6;
    const bool lead = (threadIdx.x & 63u) == 0u;
    const uint64_t row = (uint64_t)a.row0 + blockIdx.x;
    const E* const z = reinterpret_cast<const E*>(a.z) + row * a.z_stride;
    Teacher<NT> l;
    l.ask(a, row);
    float lt = wave_max(l.template take<T>(a, row, z, 0u, a.n_cols, list));
    float m = wave_max(parts_max<NT>(a, row));
    if (lead) { meet.top[0][wid] = m; meet.top[1][wid] = lt; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) { m = fmaxf(m, meet.top[0][w]); lt = fmaxf(lt, meet.top[1][w]); }
    const float ref = m == -INFINITY ? 0.0f : m;
    l.sums(a, lt, ref, list);
    double sum = wave_sum(parts_sum<NT>(a, row, ref));
    l.sum = wave_sum(l.sum);
    l.cross = wave_sum(l.cross);
    if (lead) { meet.sum[0][wid] = sum; meet.sum[1][wid] = l.sum; meet.sum[2][wid] = l.cross; }
    __syncthreads();
    sum = l.sum = l.cross = 0.0;
#pragma unroll
    for (int w = 0; w < NW; ++w) { sum += meet.sum[0][w]; l.sum += meet.sum[1][w]; l.cross += meet.sum[2][w]; }
    l.finish();
    if (threadIdx.x == 0) write_row(a, row, m, sum, l);
}

// the gradient of one chunk of one row, from the row's saved norm, or (JOIN) from its chunks' parts, joined by every workgroup
// anew; a row's first chunk then writes the row's loss and norm
template <typename T, int NT, bool JOIN>
__global__ void __launch_bounds__(NT) distill_grad_kernel(const DistillArgs a) {
    typedef typename T::elem E;
    constexpr int NW = NT / 64;
    __shared__ Meet<NW> meet;
    extern __shared__ uint32_t lds[];
    const List list(a, lds);
    const uint32_t wid = threadIdx.x >> 6;
    const bool lead = (threadIdx.x & 63u) == 0u;
    const uint64_t part = (uint64_t)a.row0 * a.n_chunks + blockIdx.x, row = part / a.n_chunks;
    const uint32_t c0 = (uint32_t)((part % a.n_chunks) * a.chunk), c1 = c0 + min(a.chunk, a.n_cols - c0);
    const E* const z = reinterpret_cast<const E*>(a.z) + row * a.z_stride;
    E* const g = reinterpret_cast<E*>(a.grad) + row * a.grad_stride;
    Teacher<NT> l;
    l.ask(a, row);
    const uint32_t whole = c0 + (c1 - c0) / T::W * T::W, ct = whole + threadIdx.x;
    const bool tail = threadIdx.x < (uint32_t)T::W && ct < c1;
    typename T::vec h[PART_VECS];
    float et = 0.0f;
#pragma unroll
    for (int v = 0; v < PART_VECS; ++v) {
        const uint32_t c = ((uint32_t)v * NT + threadIdx.x) * T::W;
        h[v] = fill_vec<T>(0.0f);
        if (c < whole - c0) h[v] = load_vec<T>(z + c0 + c);
    }
    if (tail) et = (float)z[ct];
    l.clear(a, list);
    float lt = wave_max(l.template take<T>(a, row, z, c0, c1, list));
    float m = JOIN ? wave_max(parts_max<NT>(a, row)) : a.norm_in[2 * row];
    if (lead) { meet.top[0][wid] = m; meet.top[1][wid] = lt; }
    __syncthreads();   // (everything has been read before anything is overwritten)
#pragma unroll
    for (int w = 0; w < NW; ++w) { m = fmaxf(m, meet.top[0][w]); lt = fmaxf(lt, meet.top[1][w]); }
    const float ref = m == -INFINITY ? 0.0f : m;
    l.enter(a, list, c0, c1);
    l.sums(a, lt, 0.0f, list);
    double sum = JOIN ? wave_sum(parts_sum<NT>(a, row, ref)) : 0.0;
    l.sum = wave_sum(l.sum);
    if (lead) { meet.sum[0][wid] = sum; meet.sum[1][wid] = l.sum; }
    __syncthreads();
    sum = l.sum = 0.0;
#pragma unroll
    for (int w = 0; w < NW; ++w) { sum += meet.sum[0][w]; l.sum += meet.sum[1][w]; }
    l.finish();
    const float per_sum = JOIN ? (float)(1.0 / sum) : (float)exp(-(double)a.norm_in[2 * row + 1]);
    const float gt = a.temperature * (a.weight ? a.weight[row] : 1.0f);
    const float f = gt * per_sum;
#pragma unroll
    for (int v = 0; v < PART_VECS; ++v) {
        const uint32_t c = ((uint32_t)v * NT + threadIdx.x) * T::W;
        typename T::vec o;
#pragma unroll
        for (int i = 0; i < T::W; ++i) o[i] = T::round(l.some ? f * exp2_hw(expo(a, (float)h[v][i], ref)) : 0.0f);
        if (c < whole - c0) store_vec<T>(g + c0 + c, o);
    }
    if (tail) g[ct] = T::round(l.some ? f * exp2_hw(expo(a, et, ref)) : 0.0f);
    // what the workgroup has written so far is in memory, in front of what follows
    __threadfence_block();
    __syncthreads();
    if (l.some) l.template patch<T>(a, list, g, c0, c1, ref, per_sum, gt);
    if constexpr (JOIN) {
        if (c0 == 0 && threadIdx.x == 0) {
            const float* const from = list_part(a, row);
            const uint64_t bits = (uint64_t)__builtin_bit_cast(uint32_t, from[0]) | (uint64_t)__builtin_bit_cast(uint32_t, from[1]) << 32;
            l.cross = __builtin_bit_cast(double, bits) - ((double)from[2] - (double)ref) * l.sum;
            write_row(a, row, m, sum, l);
        }
    }
}

// One workgroup a row, or a chunk of one, and a launch for every 2^20 of them (a kernel without a loop over rows keeps nothing
// from one row to the next in registers, NV = 16 with the gradient 112 of them instead of 167).
template <typename F>
void for_rows(DistillArgs a, uint64_t groups_a_row, F&& launch) {
    const uint32_t run = (uint32_t)(groups_a_row >= (1u << 20) ? 1u : (1u << 20) / groups_a_row);
    for (uint64_t row = 0; row < a.n_rows; row += run) {
        a.row0 = (uint32_t)row;
        launch(a, dim3((uint32_t)(std::min<uint64_t>(run, a.n_rows - row) * groups_a_row)));
    }
}

static_assert(F32by8::W == 8 && F16::W == 8 && BF16::W == 8 && PART_MAX % PART_STEP == 0, "a chunk fits the part kernels' registers");

// Chunks of a long row: long ones where there are rows enough to fill the chip, short ones for few rows.
uint32_t chunk_of(uint64_t n_rows, uint32_t n_cols) {
    const uint64_t want = n_rows * n_cols / 2048u;
    const uint64_t c = (want + PART_STEP - 1) / PART_STEP * PART_STEP;
    return (uint32_t)(c < PART_STEP ? PART_STEP : (c > PART_MAX ? PART_MAX : c));
}

void set_chunks(DistillArgs& a) {
    a.chunk = chunk_of(a.n_rows, a.n_cols);
    a.n_chunks = (uint32_t)(((uint64_t)a.n_cols + a.chunk - 1) / a.chunk);
}

template <typename T, int NT, int NV>
void launch_row(const DistillArgs& args, hipStream_t st) {
    for_rows(args, 1, [&](const DistillArgs& a, dim3 grid) {
        if (a.grad) hipLaunchKernelGGL((distill_row_kernel<T, NT, NV, true>), grid, dim3(NT), list_bytes(a, true), st, a);
        else hipLaunchKernelGGL((distill_row_kernel<T, NT, NV, false>), grid, dim3(NT), list_bytes(a, false), st, a);
    });
}

template <typename T, bool JOIN>
void launch_grad(const DistillArgs& args, hipStream_t st) {
    for_rows(args, args.n_chunks, [&](const DistillArgs& a, dim3 grid) {
        hipLaunchKernelGGL((distill_grad_kernel<T, 256, JOIN>), grid, dim3(256), list_bytes(a, true), st, a);
    });
}

template <typename T>
void launch_loss(DistillArgs a, hipStream_t st) {
    if (a.n_cols <= ROW_MAX) {
        // The fewest threads that hold the row, where there are rows enough to fill the chip (with the gradient, us: 5000 x 2000 bf16
        // one wave a row 15.8, two 16.9, four 20.4; 5000 x 4000 two waves 23.3, one 23.4, four 26.1; 5000 x 8000 four waves 37.6, two
        // 43.6, eight 45.8; 4096 x 20000 four waves 69, eight 79); few rows of two vectors a thread (64 x 4000 four waves 6.6, two
        // 6.9, one 7.9). The types share the rule, which costs f32 7 % at 5000 x 4000 (two waves 43.8, four 41.0), and it stops short of
        // eight waves for rows of 8193 to 32768 columns, which are faster where there are few (1 x 30000 8.7 us, eight waves 7.8; 64 x 30000
        // 9.6, 8.6; 300 x 16000 10.5, 10.2; 2000 x 16000 the same) and at 5000 x 16000 (72, 66).
        const bool many = a.n_rows >= 1024u;
        // (Very many rows of nearly what four waves hold: as 16-bit rows of eight waves three of them are on a CU at a time instead of
        // four, and reads and writes get in each other's way less. 4096 x 32000 bf16 with the gradient 104 us, four waves 111;
        // 8192 x 32000 191, 215; but 2000 x 29999 64, 60 and 4096 x 20000 79, 69. Both bounds lie between measured sizes.)
        if constexpr (sizeof(typename T::elem) == 2)
            if (a.n_cols > 24576u && a.n_cols <= 32768u && a.n_rows >= 2560u) return launch_row<T, 512, 8>(a, st);
        if (a.n_cols <= 512u) launch_row<T, 64, 1>(a, st);
        else if (a.n_cols <= 1024u) launch_row<T, 64, 2>(a, st);
        else if (a.n_cols <= 2048u && many) launch_row<T, 64, 4>(a, st);
        else if (a.n_cols <= 2048u) launch_row<T, 128, 2>(a, st);
        else if (a.n_cols <= 4096u && many) launch_row<T, 128, 4>(a, st);
        else if (a.n_cols <= 4096u) launch_row<T, 256, 2>(a, st);
        else if (a.n_cols <= 8192u) launch_row<T, 256, 4>(a, st);
        else if (a.n_cols <= 16384u) launch_row<T, 256, 8>(a, st);
        else if (a.n_cols <= 32768u) launch_row<T, 256, 16>(a, st);
        else launch_row<T, 512, 16>(a, st);
        return;
    }
    // Parts and gradient, whose workgroups join the parts in passing while there are few of them (us: 9 x 686339 bf16 16.8, with a
    // launch for the joining 18.9; 64 x 300000 27.7, 30.6; 1000 x 152064 189, 193; 1000 parts a row take the same time either way).
    if (a.grad && a.n_chunks <= JOIN_MAX) {
        for_rows(a, a.n_chunks, [&](const DistillArgs& a, dim3 grid) {
            hipLaunchKernelGGL((distill_part_kernel<T, 256, true>), grid, dim3(256), list_bytes(a, false), st, a);
        });
        return launch_grad<T, true>(a, st);
    }
    for_rows(a, a.n_chunks, [&](const DistillArgs& a, dim3 grid) { hipLaunchKernelGGL((distill_part_kernel<T, 256, false>), grid, dim3(256), 0, st, a); });
    for_rows(a, 1, [&](const DistillArgs& a, dim3 grid) { hipLaunchKernelGGL((distill_join_kernel<T, 256>), grid, dim3(256), list_bytes(a, false), st, a); });
    if (a.grad) {
        a.norm_in = a.norm;
        launch_grad<T, false>(a, st);
    }
}

uint64_t work_bytes(uint32_t n_rows, uint32_t n_cols) {
    if (n_cols <= ROW_MAX || n_rows == 0) return 0;
    const uint32_t chunk = chunk_of(n_rows, n_cols);
    return (uint64_t)n_rows * ((((uint64_t)n_cols + chunk - 1) / chunk) * 2u + 4u) * sizeof(float);
}

trag_status check_distill(const std::string& who, const DistillArgs& a, uint32_t dtype) {
    auto bad = [&](const char* what) { return set_error(TRAG_INVALID_ARG, who + ": " + what); };
    if (dtype > TRAG_BF16) return bad("unknown element type");
    if (a.n_cols == 0) return bad("rows of 0 columns");
    if (!a.z || (a.k && (!a.ids || !a.teacher))) return bad("null array");
    // (and its reciprocal finite in 32 bits, which leaves out temperatures below 5e-39; a difference of two logits is an infinity in
    // 32 bits from 3.4e38 on, whose exponential over a temperature of 1e36 is 0 as it should be, and over 1e38 e^-3.4)
    if (!(a.temperature > 0.0f) || !(a.temperature <= 1e36f) || !(a.c - a.c == 0.0f))
        return bad("the temperature must be positive, and neither below 5e-39 nor above 1e36");
    const uint32_t e = dtype_bytes(dtype);
    if (!aligned_to(a.z, e) || !aligned_to(a.grad, e) || !aligned_to(a.ids, 4) || !aligned_to(a.teacher, 4) ||
        !aligned_to(a.counts, 4) || !aligned_to(a.loss, 4) || !aligned_to(a.norm, 4) || !aligned_to(a.norm_in, 4) ||
        !aligned_to(a.weight, 4) || !aligned_to(a.parts, 4))
        return bad("an array is not aligned to its elements");
    if (a.z_stride < a.n_cols || (a.grad && a.grad_stride < a.n_cols)) return bad("a row stride is less than the number of columns");
    if (a.grad && a.grad == a.z && a.grad_stride != a.z_stride) return bad("a gradient in place of the logits needs their stride");
    if (a.k > LIST_MAX) return set_error(TRAG_UNSUPPORTED, who + ": a teacher's list is longer than 1024 entries");
    return TRAG_OK;
}

DistillArgs distill_args(const void* z, uint64_t z_stride, uint32_t n_rows, uint32_t n_cols, const uint32_t* ids,
                         const float* teacher, const uint32_t* counts, uint32_t k, float temperature) {
    DistillArgs a{};
    a.z = z; a.z_stride = z_stride; a.n_rows = n_rows; a.n_cols = n_cols;
    a.ids = ids; a.teacher = teacher; a.counts = counts; a.k = k; a.temperature = temperature;
    a.c64 = 1.4426950408889634 / (double)temperature;
    a.c = (float)a.c64;
    if (n_rows && n_cols) set_chunks(a);
    uint32_t slots = 64;
    while (slots < 2u * k && slots < 2u * LIST_MAX) slots *= 2u;
    a.slot_mask = slots - 1u;
    return a;
}

}  // namespace
}  // namespace trag

extern "C" {

uint64_t trag_distill_work_bytes(uint32_t n_rows, uint32_t n_cols) { return trag::work_bytes(n_rows, n_cols); }

trag_status trag_distill_loss_device(const void* d_logits, uint64_t logits_stride, uint32_t dtype, uint32_t n_rows,
                                     uint32_t n_cols, const uint32_t* d_ids, const float* d_teacher,
                                     const uint32_t* d_counts, uint32_t k, float temperature, float* d_loss,
                                     float* d_norm, const float* d_row_weight, void* d_grad, uint64_t grad_stride,
                                     void* d_work, uint64_t work_bytes, void* hip_stream) {
    using namespace trag;
    return op_entry([&]() -> trag_status {
        const char* who = "trag_distill_loss_device";
        if (n_rows == 0) return TRAG_OK;
        DistillArgs a = distill_args(d_logits, logits_stride, n_rows, n_cols, d_ids, d_teacher, d_counts, k, temperature);
        a.loss = d_loss; a.norm = d_norm; a.weight = d_row_weight; a.grad = d_grad; a.grad_stride = grad_stride;
        a.parts = reinterpret_cast<float*>(d_work);
        trag_status ts = check_distill(who, a, dtype);
        if (ts != TRAG_OK) return ts;
        if (!d_loss || !d_norm) return set_error(TRAG_INVALID_ARG, std::string(who) + ": null output array");
        const uint64_t need = trag::work_bytes(n_rows, n_cols);
        if (need && (!d_work || work_bytes < need))
            return set_error(TRAG_INVALID_ARG, std::string(who) + ": needs a workspace of " + std::to_string(need) + " bytes");
        OpDevice on(who, hip_stream, {d_logits, d_ids, d_teacher, d_counts, d_loss, d_norm, d_row_weight, d_grad, need ? d_work : nullptr});
        if (on.status != TRAG_OK) return on.status;
        const hipStream_t st = (hipStream_t)hip_stream;
        if (dtype == TRAG_F32) launch_loss<F32by8>(a, st);
        else if (dtype == TRAG_F16) launch_loss<F16>(a, st);
        else launch_loss<BF16>(a, st);
        return op_launched(who);
    });
}

trag_status trag_distill_grad_device(const void* d_logits, uint64_t logits_stride, uint32_t dtype, uint32_t n_rows,
                                     uint32_t n_cols, const uint32_t* d_ids, const float* d_teacher,
                                     const uint32_t* d_counts, uint32_t k, float temperature, const float* d_norm,
                                     const float* d_row_weight, void* d_grad, uint64_t grad_stride, void* hip_stream) {
    using namespace trag;
    return op_entry([&]() -> trag_status {
        const char* who = "trag_distill_grad_device";
        if (n_rows == 0) return TRAG_OK;
        DistillArgs a = distill_args(d_logits, logits_stride, n_rows, n_cols, d_ids, d_teacher, d_counts, k, temperature);
        a.norm_in = d_norm; a.weight = d_row_weight; a.grad = d_grad; a.grad_stride = grad_stride;
        trag_status ts = check_distill(who, a, dtype);
        if (ts != TRAG_OK) return ts;
        if (!d_norm || !d_grad) return set_error(TRAG_INVALID_ARG, std::string(who) + ": null array");
        OpDevice on(who, hip_stream, {d_logits, d_ids, d_teacher, d_counts, d_norm, d_row_weight, d_grad});
        if (on.status != TRAG_OK) return on.status;
        const hipStream_t st = (hipStream_t)hip_stream;
        if (dtype == TRAG_F32) launch_grad<F32by8, false>(a, st);
        else if (dtype == TRAG_F16) launch_grad<F16, false>(a, st);
        else launch_grad<BF16, false>(a, st);
        return op_launched(who);
    });
}

}  // extern "C"
