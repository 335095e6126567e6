// Distillation from a teacher's best k: Kullback-Leibler loss of rows of logits, and its gradient.
//
// A row's teacher is a list of k (column, score) pairs -- what an exact search leaves in device memory --
// with p = softmax(t / T) over the list; the student is q = softmax(z / T) over all columns.
//
//   loss = T^2 sum_j p_j (log p_j - log q_{id_j}),      d loss / d z_c = T (q_c - sum_{j: id_j = c} p_j).
//
// The loss needs two numbers of the whole row, m = max z and ln sum exp((z - m) / T), and k logits; the
// gradient needs the row again. Bound by HBM: one read of the logits for the loss, one read and one write
// for a gradient. Rows of up to 32768 columns stay in registers between the sum and the gradient (as
// exponentials, so nothing is computed twice); longer rows are cut into chunks whose partial (m, sum)
// pairs are joined by a second launch, which also fills the chip when there are few rows.
//
// Exponentials go through exp2 of (z - m) log2(e) / T: the difference first, so that rows at the type's lowest
// value, whose product with 1 / T would overflow, still come out as the distribution they are. Sums over a
// row are 32-bit per thread and chunk, 64-bit across them; the k terms of the loss are 64-bit.
#include "trag_ops.h"

namespace trag {
namespace {

constexpr uint32_t LIST_MAX = 1024;        // teacher entries per row
constexpr uint32_t ROW_MAX = 32768;        // columns of the row kernel
constexpr uint32_t PART_STEP = 2048;       // a chunk of a long row is a multiple of this
constexpr uint32_t PART_MAX = 16384;

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
    float* parts;             // 2 per row and chunk
    uint64_t z_stride, grad_stride;
    uint32_t n_rows, n_cols, k, chunk, n_chunks;
    float temperature, c;     // c = log2(e) / T
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// exponent of e^((z - m) / T) as a power of two (off by three roundings, 3 * 2^-24 relative; an infinite z stays what it is)
__device__ __forceinline__ float expo(const DistillArgs& a, float z, float m) { return (z - m) * a.c; }

template <int NW>
__device__ __forceinline__ float wg_max(float v, float* sh) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    if (NW == 1) return v;
    if ((threadIdx.x & 63u) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) v = fmaxf(v, sh[i]);
    return v;
}

template <int NW>
__device__ __forceinline__ double wg_sum(double v, double* sh) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if (NW == 1) return v;
    if ((threadIdx.x & 63u) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) v += sh[i];
    return v;
}

// A row's teacher list, entry threadIdx.x + i * NT in slot i of each thread. An entry counts if it lies
// in front of the row's count and its id is a column; p is 0 for the others. `some`: the list has
// probability at all (an empty list, or one of minus infinities, leaves the row out: loss and gradient 0).
template <int NT>
struct TeacherList {
    static constexpr int NL = (int)(LIST_MAX + NT - 1) / NT;
    uint32_t id[NL];
    float t[NL];
    double p[NL], logp[NL];
    bool there[NL];
    bool some;

    __device__ __forceinline__ void load(const DistillArgs& a, uint64_t row) {
        const uint32_t n = a.counts ? min(a.counts[row], a.k) : a.k;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t j = threadIdx.x + (uint32_t)i * NT;
            there[i] = j < n;
            id[i] = there[i] ? a.ids[row * a.k + j] : 0u;
            t[i] = there[i] ? a.teacher[row * a.k + j] : 0.0f;
            there[i] = there[i] && id[i] < a.n_cols;
        }
    }
    // sh_f, sh_d: NT / 64 words each, not shared with another reduction in between
    __device__ __forceinline__ void softmax(const DistillArgs& a, float* sh_f, double* sh_d) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < NL; ++i)
            if (there[i]) top = fmaxf(top, t[i]);   // (a NaN passes the maximum by and reaches the loss through its p)
        top = wg_max<NT / 64>(top, sh_f);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            // (a list of minus infinities: top is one, every difference would be NaN)
            logp[i] = there[i] ? ((double)t[i] - (double)(top == -INFINITY ? 0.0f : top)) / (double)a.temperature : -INFINITY;
            p[i] = there[i] ? exp(logp[i]) : 0.0;
            sum += p[i];
        }
        sum = wg_sum<NT / 64>(sum, sh_d);
        some = !(sum == 0.0);
        const double ls = some ? log(sum) : 0.0;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            logp[i] -= ls;
            p[i] = some ? p[i] / sum : 0.0;
        }
    }
};

// The gradient at the list's columns, after everything else of [c0, c1) has been written: the first entry of
// an id takes the probabilities of all entries of that id. zl: the logits there, read before they may have been
// overwritten (the gradient may go in place of the logits).
template <typename T, int NT>
__device__ __forceinline__ void patch_list(const DistillArgs& a, const TeacherList<NT>& l, const float (&zl)[TeacherList<NT>::NL],
                                           typename T::elem* g, uint32_t c0, uint32_t c1, float m, float log2sum, float gt,
                                           uint32_t* sh_id, float* sh_p) {
#pragma unroll
    for (int i = 0; i < TeacherList<NT>::NL; ++i) {
        const uint32_t j = threadIdx.x + (uint32_t)i * NT;
        if (j < a.k) { sh_id[j] = l.there[i] ? l.id[i] : 0xFFFFFFFFu; sh_p[j] = (float)l.p[i]; }
    }
    // what the workgroup has written so far is in memory, in front of what follows
    __threadfence_block();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TeacherList<NT>::NL; ++i) {
        const uint32_t j = threadIdx.x + (uint32_t)i * NT;
        if (j >= a.k || !l.there[i] || l.id[i] < c0 || l.id[i] >= c1) continue;
        bool first = true;
        for (uint32_t o = 0; o < j; ++o) first = first && sh_id[o] != l.id[i];
        if (!first) continue;
        float p = 0.0f;
        for (uint32_t o = j; o < a.k; ++o)
            if (sh_id[o] == l.id[i]) p += sh_p[o];
        const float q = exp2_hw(expo(a, zl[i], m) - log2sum);
        T::store(g + l.id[i], gt * (q - p));
    }
}

// One workgroup a row, the row in registers: NV vectors of eight columns a thread.
template <typename T, int NT, int NV, bool GRAD>
__global__ void __launch_bounds__(NT) distill_row_kernel(const DistillArgs a) {
    typedef typename T::elem E;
    constexpr int NW = NT / 64, NL = TeacherList<NT>::NL;
    __shared__ float sh_f[2][NW];
    __shared__ double sh_d[3][NW];
    __shared__ uint32_t sh_id[GRAD ? LIST_MAX : 1];
    __shared__ float sh_p[GRAD ? LIST_MAX : 1];
    for (uint64_t row = blockIdx.x; row < a.n_rows; row += gridDim.x) {
        const E* const z = reinterpret_cast<const E*>(a.z) + row * a.z_stride;
        float e[NV][8];
        float m = -INFINITY;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const uint32_t c = ((uint32_t)v * NT + threadIdx.x) * 8u;
            if (c + 8u <= a.n_cols) T::load8(z + c, e[v]);
            else {
#pragma unroll
                for (int i = 0; i < 8; ++i) e[v][i] = c + (uint32_t)i < a.n_cols ? T::load(z + c + i) : -INFINITY;
            }
        }
        TeacherList<NT> l;
        l.load(a, row);
        float zl[NL];
#pragma unroll
        for (int i = 0; i < NL; ++i) zl[i] = l.there[i] ? T::load(z + l.id[i]) : 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, e[v][i]);
        m = wg_max<NW>(m, sh_f[0]);
        const float ref = m == -INFINITY ? 0.0f : m;
        float s = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                e[v][i] = exp2_hw(expo(a, e[v][i], ref));
                s += e[v][i];
            }
        const double sum = wg_sum<NW>((double)s, sh_d[0]);
        l.softmax(a, sh_f[1], sh_d[1]);
        const double ln = log(sum);
        double part = 0.0;
#pragma unroll
        for (int i = 0; i < NL; ++i)
            if (l.there[i] && !(l.p[i] == 0.0))
                part += l.p[i] * (l.logp[i] - ((double)zl[i] - (double)ref) / (double)a.temperature + ln);
        part = wg_sum<NW>(part, sh_d[2]);
        if (threadIdx.x == 0) {
            a.loss[row] = l.some ? (float)((double)a.temperature * (double)a.temperature * part) : 0.0f;
            a.norm[2 * row] = m;
            a.norm[2 * row + 1] = (float)ln;
        }
        if constexpr (GRAD) {
            E* const g = reinterpret_cast<E*>(a.grad) + row * a.grad_stride;
            const float gt = a.temperature * (a.weight ? a.weight[row] : 1.0f);
            const float f = (float)((double)gt / sum);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const uint32_t c = ((uint32_t)v * NT + threadIdx.x) * 8u;
                float o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = l.some ? e[v][i] * f : 0.0f;
                if (c + 8u <= a.n_cols) T::store8(g + c, o);
                else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (c + (uint32_t)i < a.n_cols) T::store(g + c + i, o[i]);
                }
            }
            if (l.some) patch_list<T, NT>(a, l, zl, g, 0, a.n_cols, ref, (float)(ln * 1.4426950408889634), gt, sh_id, sh_p);
        }
        __syncthreads();   // the next row's reductions and lists reuse the arrays
    }
}

// (max, sum) of one chunk of one row
template <typename T, int NT>
__global__ void __launch_bounds__(NT) distill_part_kernel(const DistillArgs a) {
    typedef typename T::elem E;
    constexpr int NW = NT / 64;
    __shared__ float sh_f[NW];
    __shared__ double sh_d[NW];
    const uint64_t n_parts = (uint64_t)a.n_rows * a.n_chunks;
    for (uint64_t part = blockIdx.x; part < n_parts; part += gridDim.x) {
        const uint64_t row = part / a.n_chunks;
        const uint64_t c0 = (part % a.n_chunks) * a.chunk, c1 = min(c0 + a.chunk, (uint64_t)a.n_cols);
        const E* const z = reinterpret_cast<const E*>(a.z) + row * a.z_stride;
        float m = -INFINITY, s = 0.0f;
        for (uint64_t c = c0 + threadIdx.x * 8u; c < c1; c += NT * 8u) {
            float e[8];
            if (c + 8u <= c1) T::load8(z + c, e);
            else {
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = c + (uint32_t)i < c1 ? T::load(z + c + i) : -INFINITY;
            }
            float top = e[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) top = fmaxf(top, e[i]);
            if (top > m) {   // (rare after the first few: the maximum of a random sequence moves ln n times)
                s = m == -INFINITY ? s : s * exp2_hw(expo(a, m, top));
                m = top;
            }
            const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += exp2_hw(expo(a, e[i], ref));
        }
        const float top = wg_max<NW>(m, sh_f);
        const float ref = top == -INFINITY ? 0.0f : top;
        const float f = m == -INFINITY ? 1.0f : exp2_hw(expo(a, m, ref));
        const double sum = wg_sum<NW>((double)s * (double)f, sh_d);
        if (threadIdx.x == 0) {
            a.parts[2 * part] = top;
            a.parts[2 * part + 1] = (float)sum;
        }
        __syncthreads();
    }
}

// a row's chunks joined, and its loss
template <typename T, int NT>
__global__ void __launch_bounds__(NT) distill_join_kernel(const DistillArgs a) {
    typedef typename T::elem E;
    constexpr int NW = NT / 64, NL = TeacherList<NT>::NL;
    __shared__ float sh_f[2][NW];
    __shared__ double sh_d[3][NW];
    for (uint64_t row = blockIdx.x; row < a.n_rows; row += gridDim.x) {
        const E* const z = reinterpret_cast<const E*>(a.z) + row * a.z_stride;
        const float* const parts = a.parts + 2 * row * a.n_chunks;
        TeacherList<NT> l;
        l.load(a, row);
        float zl[NL];
#pragma unroll
        for (int i = 0; i < NL; ++i) zl[i] = l.there[i] ? T::load(z + l.id[i]) : 0.0f;
        float m = -INFINITY;
        for (uint32_t c = threadIdx.x; c < a.n_chunks; c += NT) m = fmaxf(m, parts[2 * c]);
        m = wg_max<NW>(m, sh_f[0]);
        const float ref = m == -INFINITY ? 0.0f : m;
        double s = 0.0;
        for (uint32_t c = threadIdx.x; c < a.n_chunks; c += NT) {
            const float pm = parts[2 * c];
            // (a chunk without a number: its sum is 0, or NaN, and stays that)
            s += (double)parts[2 * c + 1] * (pm == -INFINITY ? 1.0 : (double)exp2_hw(expo(a, pm, ref)));
        }
        const double sum = wg_sum<NW>(s, sh_d[0]);
        l.softmax(a, sh_f[1], sh_d[1]);
        const double ln = log(sum);
        double part = 0.0;
#pragma unroll
        for (int i = 0; i < NL; ++i)
            if (l.there[i] && !(l.p[i] == 0.0))
                part += l.p[i] * (l.logp[i] - ((double)zl[i] - (double)ref) / (double)a.temperature + ln);
        part = wg_sum<NW>(part, sh_d[2]);
        if (threadIdx.x == 0) {
            a.loss[row] = l.some ? (float)((double)a.temperature * (double)a.temperature * part) : 0.0f;
            a.norm[2 * row] = m;
            a.norm[2 * row + 1] = (float)ln;
        }
        __syncthreads();
    }
}

// the gradient of one chunk of one row, from the row's saved norm
template <typename T, int NT>
__global__ void __launch_bounds__(NT) distill_grad_kernel(const DistillArgs a) {
    typedef typename T::elem E;
    constexpr int NW = NT / 64, NL = TeacherList<NT>::NL;
    __shared__ float sh_f[NW];
    __shared__ double sh_d[NW];
    __shared__ uint32_t sh_id[LIST_MAX];
    __shared__ float sh_p[LIST_MAX];
    const uint64_t n_parts = (uint64_t)a.n_rows * a.n_chunks;
    for (uint64_t part = blockIdx.x; part < n_parts; part += gridDim.x) {
        const uint64_t row = part / a.n_chunks;
        const uint64_t c0 = (part % a.n_chunks) * a.chunk, c1 = min(c0 + a.chunk, (uint64_t)a.n_cols);
        const E* const z = reinterpret_cast<const E*>(a.z) + row * a.z_stride;
        E* const g = reinterpret_cast<E*>(a.grad) + row * a.grad_stride;
        TeacherList<NT> l;
        l.load(a, row);
        float zl[NL];
#pragma unroll
        for (int i = 0; i < NL; ++i) zl[i] = l.there[i] && l.id[i] >= c0 && l.id[i] < c1 ? T::load(z + l.id[i]) : 0.0f;
        l.softmax(a, sh_f, sh_d);   // (its barriers also stand between the reads of zl and the writes below)
        const float m = a.norm_in[2 * row];
        const float ref = m == -INFINITY ? 0.0f : m;
        const float log2sum = (float)((double)a.norm_in[2 * row + 1] * 1.4426950408889634);
        const float gt = a.temperature * (a.weight ? a.weight[row] : 1.0f);
        for (uint64_t c = c0 + threadIdx.x * 8u; c < c1; c += NT * 8u) {
            float e[8];
            const bool full = c + 8u <= c1;
            if (full) T::load8(z + c, e);
            else {
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = c + (uint32_t)i < c1 ? T::load(z + c + i) : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = l.some ? gt * exp2_hw(expo(a, e[i], ref) - log2sum) : 0.0f;
            if (full) T::store8(g + c, e);
            else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c + (uint32_t)i < c1) T::store(g + c + i, e[i]);
            }
        }
        if (l.some) patch_list<T, NT>(a, l, zl, g, (uint32_t)c0, (uint32_t)c1, ref, log2sum, gt, sh_id, sh_p);
        __syncthreads();
    }
}

uint32_t grid_of(uint64_t n) { return (uint32_t)(n < (1u << 20) ? n : (1u << 20)); }

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
void launch_row(const DistillArgs& a, hipStream_t st) {
    if (a.grad) hipLaunchKernelGGL((distill_row_kernel<T, NT, NV, true>), dim3(grid_of(a.n_rows)), dim3(NT), 0, st, a);
    else hipLaunchKernelGGL((distill_row_kernel<T, NT, NV, false>), dim3(grid_of(a.n_rows)), dim3(NT), 0, st, a);
}

template <typename T>
void launch_grad(const DistillArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((distill_grad_kernel<T, 256>), dim3(grid_of((uint64_t)a.n_rows * a.n_chunks)), dim3(256), 0, st, a);
}

template <typename T>
void launch_loss(DistillArgs a, hipStream_t st) {
    if (a.n_cols <= ROW_MAX) {
        if (a.n_cols <= 2048u) launch_row<T, 256, 1>(a, st);
        else if (a.n_cols <= 4096u) launch_row<T, 256, 2>(a, st);
        else if (a.n_cols <= 8192u) launch_row<T, 256, 4>(a, st);
        else if (a.n_cols <= 16384u) launch_row<T, 512, 4>(a, st);
        else launch_row<T, 1024, 4>(a, st);
        return;
    }
    hipLaunchKernelGGL((distill_part_kernel<T, 256>), dim3(grid_of((uint64_t)a.n_rows * a.n_chunks)), dim3(256), 0, st, a);
    hipLaunchKernelGGL((distill_join_kernel<T, 256>), dim3(grid_of(a.n_rows)), dim3(256), 0, st, a);
    if (a.grad) {
        a.norm_in = a.norm;
        launch_grad<T>(a, st);
    }
}

uint64_t work_bytes(uint32_t n_rows, uint32_t n_cols) {
    if (n_cols <= ROW_MAX || n_rows == 0) return 0;
    const uint32_t chunk = chunk_of(n_rows, n_cols);
    return (uint64_t)n_rows * (((uint64_t)n_cols + chunk - 1) / chunk) * 2u * sizeof(float);
}

trag_status check_distill(const std::string& who, const DistillArgs& a, uint32_t dtype) {
    auto bad = [&](const char* what) { return set_error(TRAG_INVALID_ARG, who + ": " + what); };
    if (dtype > TRAG_BF16) return bad("unknown element type");
    if (a.n_cols == 0) return bad("rows of 0 columns");
    if (!a.z || (a.k && (!a.ids || !a.teacher))) return bad("null array");
    if (!(a.temperature > 0.0f) || !(a.temperature - a.temperature == 0.0f)) return bad("the temperature must be positive and finite");
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
    a.c = (float)(1.4426950408889634 / (double)temperature);
    if (n_rows && n_cols) set_chunks(a);
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
        if (dtype == TRAG_F32) launch_loss<F32>(a, st);
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
        if (dtype == TRAG_F32) launch_grad<F32>(a, st);
        else if (dtype == TRAG_F16) launch_grad<F16>(a, st);
        else launch_grad<BF16>(a, st);
        return op_launched(who);
    });
}

}  // extern "C"
