// Rows of 8-bit integers with one scale a row: from an encoder's last step (residual addition and
// root-mean-square norm) or from rows as they are (a corpus).
//
//   h = x + residual,  rms = sqrt(mean h^2 + eps),  y = h w / rms,
//   scale = max |y| / 127,  q = nearest(y / scale), ties to even.
//
// The norm cancels in q: with p = h w it is nearest(127 p / max |p|), so the integers need one maximum
// and the scale one sum, and both come out of ONE pass over the row, which stays in registers between
// the loads and the stores. p, the maximum, the sum of squares and the quotient are held in 64 bits: a
// quotient within a rounding of a border decides a whole step of the grid, and the 64-bit operations hide
// behind the memory traffic that bounds the kernel. Without them q would depend on the order of f32
// roundings; with them it is a function of the inputs alone.
//
// Bound by HBM: per element a read of x (and the residual), a write of the sum, of q and, if asked for, of
// the values they stand for. 16 lanes to a workgroup a row, by its length and how many rows there are; a row too
// long for registers (over 32768 elements) is read twice, the second time from the caches.
#include "trag_ops.h"

namespace trag {
namespace {

struct Q8Args {
    const void* x;
    const void* residual;
    const void* weight;
    void* sum;
    int8_t* q8;
    float* scale;
    void* values;
    uint64_t x_stride, residual_stride, sum_stride, q8_stride, values_stride;
    uint32_t n_rows, dim;
    float eps;
    uint32_t row0;   // first row of a launch
};

// nearest(127 p / top), ties to even. inv = 127 / top has its own rounding, which could move a tie off the
// middle (or onto it): next to a border the side is taken from 127 p against the border times top.
__device__ __forceinline__ int q8_nearest(double p, double inv, double top) {
    const double t = p * inv;
    double r = __builtin_rint(t);
    if (__builtin_fabs(__builtin_fabs(t - r) - 0.5) < 1e-9) {
        const double lo = __builtin_floor(t), c = lo + 0.5;
        const double d = __builtin_fma(p, 127.0, -(c * top));
        const double even = __builtin_rint(c);
        r = d > 0.0 ? lo + 1.0 : (d < 0.0 ? lo : even);
    }
    return (int)r;
}

// h w of N consecutive elements (W, or one behind the last whole vector); h goes to the sum's array and into the row's sum
// of squares
template <typename T, bool NORM, int N>
__device__ __forceinline__ void products(const typename T::elem* x, const typename T::elem* res, const typename T::elem* w,
                                         typename T::elem* sum, uint32_t e, double (&p)[N], double& ss) {
    typedef typename T::elem E;
    E xv[N], rv[N], wv[N];
    if constexpr (N == T::W) {
        const typename T::vec v = load_vec<T>(x + e);
#pragma unroll
        for (int i = 0; i < N; ++i) xv[i] = v[i];
        if (NORM && res) {
            const typename T::vec r = load_vec<T>(res + e);
#pragma unroll
            for (int i = 0; i < N; ++i) rv[i] = r[i];
        }
        if (NORM && w) {
            const typename T::vec u = load_vec<T>(w + e);
#pragma unroll
            for (int i = 0; i < N; ++i) wv[i] = u[i];
        }
    } else {
        xv[0] = x[e];
        if (NORM && res) rv[0] = res[e];
        if (NORM && w) wv[0] = w[e];
    }
    if (NORM && sum) {
        typename T::vec s;
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = T::round(res ? (float)xv[i] + (float)rv[i] : (float)xv[i]);
        if constexpr (N == T::W) store_vec<T>(sum + e, s);
        else sum[e] = s[0];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        double h = (double)(float)xv[i];
        if (NORM && res) h += (double)(float)rv[i];
        p[i] = (NORM && w) ? h * (double)(float)wv[i] : h;
        if (NORM) ss = __builtin_fma(h, h, ss);
        ss = __builtin_fma(p[i], 0.0, ss);   // (NaN as soon as a product is not finite; the maximum alone would pass over a NaN)
    }
}

typedef uint32_t u32_any __attribute__((aligned(1)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

template <typename T, int N>
__device__ __forceinline__ void store_q8(int8_t* q8, typename T::elem* values, uint32_t e, const double (&p)[N], double inv, double top, float scale) {
    int q[N];
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = inv > 0.0 ? q8_nearest(p[i], inv, top) : 0;
    if constexpr (N == T::W) {
        uint32_t o[N / 4];
#pragma unroll
        for (int h = 0; h < N / 4; ++h)
            o[h] = (uint32_t)(q[4 * h] & 255) | (uint32_t)(q[4 * h + 1] & 255) << 8 | (uint32_t)(q[4 * h + 2] & 255) << 16 |
                   (uint32_t)q[4 * h + 3] << 24;
        if constexpr (N == 8) *reinterpret_cast<u32x2_any*>(q8 + e) = u32x2_any{o[0], o[1]};
        else *reinterpret_cast<u32_any*>(q8 + e) = o[0];
        if (values) {
            typename T::vec v;
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = T::round((float)q[i] * scale);
            store_vec<T>(values + e, v);
        }
    } else {
        q8[e] = (int8_t)q[0];
        if (values) values[e] = T::round((float)q[0] * scale);
    }
}

template <int L>
__device__ __forceinline__ double lanes_max(double v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = __builtin_fmax(v, __shfl_xor(v, o));
    return v;
}
template <int L>
__device__ __forceinline__ double lanes_sum(double v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// From a row's maximum and sum: the factor of the integers (0: a row of zeros, or one that is not finite) and the scale.
template <bool NORM>
__device__ __forceinline__ void row_scale(const Q8Args& a, double top, double ss, double& inv, float& scale) {
    const bool fine = ss - ss == 0.0;
    inv = fine && top > 0.0 ? 127.0 / top : 0.0;
    double s = top / 127.0;
    if (NORM && top > 0.0) s /= __builtin_sqrt(ss / (double)a.dim + (double)a.eps);
    scale = fine ? (float)s : __builtin_nanf("");
}

// NT threads a row (16 lanes, a wave, or a workgroup), NV vectors of W elements a thread; the elements behind the last whole
// vector: one each for the first few threads. NV == 0: the row does not fit the registers, it is read again for the
// integers. What bounds it: 16384 x 4096 bf16 with residual, sum and values 111 us, 5.4 TB/s, what a large copy reaches. (Tried:
// the loads of all vectors ahead of the arithmetic, 81 registers instead of 58: 120 us; 4000 x 12000 118 instead of 84.)
template <typename T, bool NORM, int NT, int NV>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) q8_rows_kernel(const Q8Args a) {
    typedef typename T::elem E;
    static_assert(NT <= 64 || NT >= 256, "a row is a part of a wave, a wave or a workgroup");
    constexpr int NW = NT / 64, W = T::W;
    constexpr int L = NT < 64 ? NT : 64;                   // lanes that reduce together
    constexpr uint32_t RPB = NT < 256 ? 256u / NT : 1u;    // rows a workgroup has at a time
    __shared__ double sh[NW > 1 ? NW : 1][2];
    const uint32_t t = threadIdx.x % (NT < 256 ? NT : 1024);
    const E* const w = reinterpret_cast<const E*>(a.weight);
    const uint32_t whole = a.dim / W * W, et = whole + t;
    const bool tail = t < (uint32_t)W && et < a.dim;
    const uint64_t row = (uint64_t)a.row0 + (uint64_t)blockIdx.x * RPB + (NT < 256 ? threadIdx.x / NT : 0u);
    if (row >= a.n_rows) return;   // (parts of a wave at most: a workgroup's row is always there)
    const E* const x = reinterpret_cast<const E*>(a.x) + row * a.x_stride;
    const E* const res = a.residual ? reinterpret_cast<const E*>(a.residual) + row * a.residual_stride : nullptr;
    E* const sum = a.sum ? reinterpret_cast<E*>(a.sum) + row * a.sum_stride : nullptr;
    E* const values = a.values ? reinterpret_cast<E*>(a.values) + row * a.values_stride : nullptr;
    int8_t* const q8 = a.q8 + row * a.q8_stride;
    double top = 0.0, ss = 0.0;
    double p[NV > 0 ? NV : 1][W], pt[1] = {0.0};
    if constexpr (NV > 0) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const uint32_t e = ((uint32_t)v * NT + t) * W;
            if (e < whole) {
                products<T, NORM, W>(x, res, w, sum, e, p[v], ss);
#pragma unroll
                for (int i = 0; i < W; ++i) top = __builtin_fmax(top, __builtin_fabs(p[v][i]));
            }
        }
        if (tail) products<T, NORM, 1>(x, res, w, sum, et, pt, ss);
    } else {
        // (the sum is written in the second pass: it may go in place of an operand)
        for (uint32_t e = t * W; e < whole; e += NT * W) {
            products<T, NORM, W>(x, res, w, nullptr, e, p[0], ss);
#pragma unroll
            for (int i = 0; i < W; ++i) top = __builtin_fmax(top, __builtin_fabs(p[0][i]));
        }
        if (tail) products<T, NORM, 1>(x, res, w, nullptr, et, pt, ss);
    }
    top = __builtin_fmax(top, __builtin_fabs(pt[0]));
    top = lanes_max<L>(top);
    ss = lanes_sum<L>(ss);
    if constexpr (NW > 1) {
        if ((threadIdx.x & 63u) == 0) { sh[threadIdx.x >> 6][0] = top; sh[threadIdx.x >> 6][1] = ss; }
        __syncthreads();
        top = sh[0][0];
        ss = sh[0][1];
#pragma unroll
        for (int i = 1; i < NW; ++i) { top = __builtin_fmax(top, sh[i][0]); ss += sh[i][1]; }
    }
    double inv;
    float scale;
    row_scale<NORM>(a, top, ss, inv, scale);
    if (t == 0) a.scale[row] = scale;
    if constexpr (NV > 0) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const uint32_t e = ((uint32_t)v * NT + t) * W;
            if (e < whole) store_q8<T, W>(q8, values, e, p[v], inv, top, scale);
        }
    } else {
        double again = 0.0;
        for (uint32_t e = t * W; e < whole; e += NT * W) {
            products<T, NORM, W>(x, res, w, sum, e, p[0], again);
            store_q8<T, W>(q8, values, e, p[0], inv, top, scale);
        }
        if (tail) products<T, NORM, 1>(x, res, w, sum, et, pt, again);
    }
    if (tail) store_q8<T, 1>(q8, values, et, pt, inv, top, scale);
}

// NV: vectors of eight elements, whatever the type. A launch for every 2^20 workgroups: a kernel without a loop over rows keeps
// nothing from one row to the next in registers.
template <typename T, bool NORM, int NT, int NV>
void launch_one(const Q8Args& a, hipStream_t st) {
    constexpr uint32_t rpb = NT < 256 ? 256u / NT : 1u, run = rpb << 20;
    Q8Args r = a;
    for (uint64_t row = 0; row < a.n_rows; row += run) {
        const uint64_t rows = a.n_rows - row < run ? a.n_rows - row : run;
        r.row0 = (uint32_t)row;
        hipLaunchKernelGGL((q8_rows_kernel<T, NORM, NT, NV * 8 / T::W>), dim3((uint32_t)((rows + rpb - 1) / rpb)), dim3(NT < 256 ? 256 : NT), 0, st, r);
    }
}

template <typename T, bool NORM>
void launch_type(const Q8Args& a, hipStream_t st) {
    // Many rows: as few lanes a row as hold it -- more bytes of a lane in flight, fewer steps of the reductions -- and twice as many
    // in f32, whose vectors hold four elements. us, by lanes a row, 16-bit with the norm: 300k x 384 16 lanes 196, 32 214, 64 284;
    // 200k x 768 32 lanes 252, 64 274; 30k x 1500 64 lanes 87, 256 107; 16384 x 4096 256 threads 111, 512 137; 4000 x 12000 1024
    // threads 84, 512 86, 256 91. f32 as it is: 1M x 384 16 lanes 615, 64 600; 150k x 2048 64 lanes 507, 256 458; 60k x 4096 256
    // threads 386, 512 369.
    // Few rows: as many lanes as there is work for, since a row's time is its longest lane's (us of the kernel among others of its
    // kind, 16-bit with the norm: 1 x 384 64 lanes 2.8, 16 lanes 5.2, 1000 rows 3.5, 6.0, 6000 rows 11, 9.4; 400 x 768 256 threads
    // 4.2, 64 lanes 4.9, 32 lanes 5.9; 1000 x 2048 256 threads 8.1, 64 lanes 9.9, 2000 rows 12.5, 12.4; 1 x 6000 512 threads
    // 4.4, 256 5.1, 1000 rows 13.2, 12.9).
    const bool few = a.n_rows <= 1024u, some = a.n_rows <= 4096u;
    if constexpr (T::W == 4) {
        if (a.dim <= 128u) some ? launch_one<T, NORM, 32, 1>(a, st) : launch_one<T, NORM, 16, 1>(a, st);
        else if (a.dim <= 256u) some ? launch_one<T, NORM, 64, 1>(a, st) : launch_one<T, NORM, 32, 1>(a, st);
        else if (a.dim <= 512u) launch_one<T, NORM, 64, 1>(a, st);
        else if (a.dim <= 1024u && !few) launch_one<T, NORM, 64, 2>(a, st);
        else if (a.dim <= 2048u) launch_one<T, NORM, 256, 1>(a, st);
        else if (a.dim <= 4096u) launch_one<T, NORM, 512, 1>(a, st);
        else if (a.dim <= 8192u) launch_one<T, NORM, 512, 2>(a, st);
        else if (a.dim <= 16384u) launch_one<T, NORM, 1024, 2>(a, st);
        else if (a.dim <= 32768u) launch_one<T, NORM, 1024, 4>(a, st);
        else launch_one<T, NORM, 1024, 0>(a, st);
    } else {
        if (a.dim <= 128u) launch_one<T, NORM, 16, 1>(a, st);
        else if (a.dim <= 256u) some ? launch_one<T, NORM, 32, 1>(a, st) : launch_one<T, NORM, 16, 2>(a, st);
        else if (a.dim <= 512u && some) launch_one<T, NORM, 64, 1>(a, st);
        else if (a.dim <= 384u) launch_one<T, NORM, 16, 3>(a, st);
        else if (a.dim <= 512u) launch_one<T, NORM, 32, 2>(a, st);
        else if (a.dim <= 2048u && few) launch_one<T, NORM, 256, 1>(a, st);
        else if (a.dim <= 768u && a.n_rows > 2048u) launch_one<T, NORM, 32, 3>(a, st);
        else if (a.dim <= 1024u) launch_one<T, NORM, 64, 2>(a, st);
        else if (a.dim <= 1536u) launch_one<T, NORM, 64, 3>(a, st);
        else if (a.dim <= 2048u) launch_one<T, NORM, 64, 4>(a, st);
        else if (a.dim <= 4096u) launch_one<T, NORM, 256, 2>(a, st);
        else if (a.dim <= 8192u) a.n_rows <= 512u ? launch_one<T, NORM, 512, 2>(a, st) : launch_one<T, NORM, 256, 4>(a, st);
        else if (a.dim <= 16384u) launch_one<T, NORM, 1024, 2>(a, st);
        else if (a.dim <= 32768u) launch_one<T, NORM, 1024, 4>(a, st);
        else launch_one<T, NORM, 1024, 0>(a, st);
    }
}

template <bool NORM>
void launch_q8(const Q8Args& a, uint32_t dtype, hipStream_t st) {
    if (dtype == TRAG_F32) launch_type<F32, NORM>(a, st);
    else if (dtype == TRAG_F16) launch_type<F16, NORM>(a, st);
    else launch_type<BF16, NORM>(a, st);
}

trag_status check_rows(const std::string& who, const Q8Args& a, uint32_t dtype) {
    auto bad = [&](const char* what) { return set_error(TRAG_INVALID_ARG, who + ": " + what); };
    if (dtype > TRAG_BF16) return bad("unknown element type");
    if (a.dim == 0) return bad("dim is 0");
    if (a.dim > (1u << 30)) return set_error(TRAG_UNSUPPORTED, who + ": dim is more than 2^30");
    if (!a.x || !a.q8 || !a.scale) return bad("null array");
    const uint32_t e = dtype_bytes(dtype);
    if (!aligned_to(a.x, e) || !aligned_to(a.residual, e) || !aligned_to(a.weight, e) || !aligned_to(a.sum, e) ||
        !aligned_to(a.values, e) || !aligned_to(a.scale, 4))
        return bad("an array is not aligned to its elements");
    if (a.x_stride < a.dim || (a.residual && a.residual_stride < a.dim) || (a.sum && a.sum_stride < a.dim) ||
        a.q8_stride < a.dim || (a.values && a.values_stride < a.dim))
        return bad("a row stride is less than dim");
    // in place means the same rows: every thread reads what it later overwrites, nobody else does
    if ((a.sum == a.x && a.sum && a.sum_stride != a.x_stride) || (a.sum && a.sum == a.residual && a.sum_stride != a.residual_stride) ||
        (a.values && a.values == a.x && a.values_stride != a.x_stride) ||
        (a.values && a.values == a.residual && a.values_stride != a.residual_stride))
        return bad("an output in place of an input needs the input's stride");
    if (a.values && a.values == a.sum) return bad("the sum and the values cannot share an array");
    return TRAG_OK;
}

}  // namespace

hipError_t launch_quantize_rows_f32(const float* d_rows, uint64_t stride, uint32_t n_rows, uint32_t dim, int8_t* d_q8,
                                    uint64_t q8_stride, float* d_scale, hipStream_t st) {
    Q8Args a{};
    a.x = d_rows; a.x_stride = stride;
    a.q8 = d_q8; a.q8_stride = q8_stride; a.scale = d_scale;
    a.n_rows = n_rows; a.dim = dim;
    launch_q8<false>(a, TRAG_F32, st);
    return hipGetLastError();
}

}  // namespace trag

extern "C" {

trag_status trag_rmsnorm_q8_device(const void* d_x, uint64_t x_stride, const void* d_residual, uint64_t residual_stride,
                                   const void* d_weight, float eps, uint32_t dtype, uint32_t n_rows, uint32_t dim,
                                   void* d_sum, uint64_t sum_stride, int8_t* d_q8, uint64_t q8_stride, float* d_scale,
                                   void* d_values, uint64_t values_stride, void* hip_stream) {
    using namespace trag;
    return op_entry([&]() -> trag_status {
        const char* who = "trag_rmsnorm_q8_device";
        if (n_rows == 0) return TRAG_OK;
        const Q8Args a{d_x, d_residual, d_weight, d_sum, d_q8, d_scale, d_values, x_stride, residual_stride, sum_stride,
                       q8_stride, values_stride, n_rows, dim, eps, 0};
        trag_status ts = check_rows(who, a, dtype);
        if (ts != TRAG_OK) return ts;
        if (!(eps >= 0.0f) || !(eps - eps == 0.0f)) return set_error(TRAG_INVALID_ARG, std::string(who) + ": eps must be finite and not negative");
        OpDevice on(who, hip_stream, {d_x, d_residual, d_weight, d_sum, d_q8, d_scale, d_values});
        if (on.status != TRAG_OK) return on.status;
        launch_q8<true>(a, dtype, (hipStream_t)hip_stream);
        return op_launched(who);
    });
}

trag_status trag_quantize_q8_device(const void* d_x, uint64_t x_stride, uint32_t dtype, uint32_t n_rows, uint32_t dim,
                                    int8_t* d_q8, uint64_t q8_stride, float* d_scale, void* d_values,
                                    uint64_t values_stride, void* hip_stream) {
    using namespace trag;
    return op_entry([&]() -> trag_status {
        const char* who = "trag_quantize_q8_device";
        if (n_rows == 0) return TRAG_OK;
        const Q8Args a{d_x, nullptr, nullptr, nullptr, d_q8, d_scale, d_values, x_stride, 0, 0, q8_stride, values_stride,
                       n_rows, dim, 0.0f, 0};
        trag_status ts = check_rows(who, a, dtype);
        if (ts != TRAG_OK) return ts;
        OpDevice on(who, hip_stream, {d_x, d_q8, d_scale, d_values});
        if (on.status != TRAG_OK) return on.status;
        launch_q8<false>(a, dtype, (hipStream_t)hip_stream);
        return op_launched(who);
    });
}

}  // extern "C"
