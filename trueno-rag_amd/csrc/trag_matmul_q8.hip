// Product of rows of 8-bit integers, each with its scale: out[i][j] = (sum_k a[i][k] b[j][k]) sa[i] sb[j].
// Queries against a corpus, tokens against a linear layer's channels.
//
// The sum is an integer: exact in 32 bits up to 131071 terms (128 * 128 * 131071 < 2^31), whatever the
// order, so every form of the kernel gives the same bits. It is rounded once to f32, multiplied by the two
// scales (one rounding each) and rounded to the output's type.
#include "trag_ops.h"

namespace trag {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v4i_any __attribute__((ext_vector_type(4), aligned(1)));

constexpr uint32_t DIM_MAX = 131071;

struct MmArgs {
    const int8_t* a;
    const int8_t* b;
    const float* sa;
    const float* sb;
    void* out;
    uint64_t lda, ldb, ldo;
    uint32_t m, n, dim;
};

// 16 bytes of a row from k on, zeros behind its end (a zero on both sides adds nothing)
__device__ __forceinline__ v4i load_row16(const int8_t* row, uint32_t k, uint32_t dim) {
    if (k + 16u <= dim) return *reinterpret_cast<const v4i_any*>(row + k);
    v4i r = {0, 0, 0, 0};
    if (k < dim) {
#pragma unroll
        for (uint32_t i = 0; i < 16u; ++i)
            if (k + i < dim) r[i >> 2] |= (int)((uint32_t)(uint8_t)row[k + i] << (8u * (i & 3u)));
    }
    return r;
}

__device__ __forceinline__ float scaled(int acc, float sa, float sb) { return (float)acc * sa * sb; }

// Any alignment, any width: 128 x 128 tile, four waves of 64 x 64, operands through registers into LDS.
// A row of LDS is 80 bytes: the 16 rows of a fragment read start on 16 different groups of four banks.
template <typename T>
__global__ void __launch_bounds__(256) mm_any_kernel(const MmArgs p) {
    typedef typename T::elem E;
    constexpr int LD = 80;
    __shared__ __attribute__((aligned(16))) int8_t As[128 * LD];
    __shared__ __attribute__((aligned(16))) int8_t Bs[128 * LD];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wid = tid >> 6;
    const uint32_t m_tiles = (p.m + 127u) / 128u;
    const uint32_t mt = blockIdx.x % m_tiles, nt = blockIdx.x / m_tiles;
    const uint32_t m0 = mt * 128u, n0 = nt * 128u;
    const uint32_t wm = (wid >> 1) * 64u, wn = (wid & 1u) * 64u;
    const int8_t *ar[2], *br[2];
    uint32_t kc[2], slot[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t c = tid + (uint32_t)i * 256u, r = c >> 2;
        kc[i] = (c & 3u) * 16u;
        slot[i] = r * LD + kc[i];
        ar[i] = p.a + (uint64_t)min(m0 + r, p.m - 1u) * p.lda;
        br[i] = p.b + (uint64_t)min(n0 + r, p.n - 1u) * p.ldb;
    }
    v4i acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = v4i{0, 0, 0, 0};
    v4i fa[2], fb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) { fa[i] = load_row16(ar[i], kc[i], p.dim); fb[i] = load_row16(br[i], kc[i], p.dim); }
    for (uint32_t k0 = 0; k0 < p.dim; k0 += 64u) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            *reinterpret_cast<v4i*>(As + slot[i]) = fa[i];
            *reinterpret_cast<v4i*>(Bs + slot[i]) = fb[i];
        }
        __syncthreads();
        if (k0 + 64u < p.dim) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = load_row16(ar[i], k0 + 64u + kc[i], p.dim);
                fb[i] = load_row16(br[i], k0 + 64u + kc[i], p.dim);
            }
        }
        const uint32_t fr = (lane & 15u) * LD + (lane >> 4) * 16u;
        v4i xa[4], xb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            xa[i] = *reinterpret_cast<const v4i*>(As + (wm + (uint32_t)i * 16u) * LD + fr);
            xb[i] = *reinterpret_cast<const v4i*>(Bs + (wn + (uint32_t)i * 16u) * LD + fr);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xa[i], xb[j], acc[i][j], 0, 0, 0);
    }
    // lane l holds column l % 16 of rows 4 (l / 16) .. + 3
    E* const out = reinterpret_cast<E*>(p.out);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t col = n0 + wn + (uint32_t)j * 16u + (lane & 15u);
        const float sb = col < p.n ? (p.sb ? p.sb[col] : 1.0f) : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t row = m0 + wm + (uint32_t)i * 16u + (lane >> 4) * 4u + (uint32_t)r;
                if (row < p.m && col < p.n) T::store(out + (uint64_t)row * p.ldo + col, scaled(acc[i][j][r], p.sa ? p.sa[row] : 1.0f, sb));
            }
    }
}

template <typename T>
void launch_mm(const MmArgs& p, hipStream_t st) {
    const uint64_t tiles = (uint64_t)((p.m + 127u) / 128u) * ((p.n + 127u) / 128u);
    hipLaunchKernelGGL((mm_any_kernel<T>), dim3((uint32_t)tiles), dim3(256), 0, st, p);
}

}  // namespace
}  // namespace trag

extern "C" trag_status trag_matmul_q8_device(const int8_t* d_a, uint64_t a_stride, const float* d_a_scale, const int8_t* d_b,
                                             uint64_t b_stride, const float* d_b_scale, uint32_t m, uint32_t n, uint32_t dim,
                                             uint32_t out_dtype, void* d_out, uint64_t out_stride, void* hip_stream) {
    using namespace trag;
    return op_entry([&]() -> trag_status {
        const char* who = "trag_matmul_q8_device";
        auto bad = [&](const char* what) { return set_error(TRAG_INVALID_ARG, std::string(who) + ": " + what); };
        if (m == 0 || n == 0) return TRAG_OK;
        if (out_dtype > TRAG_BF16) return bad("unknown element type");
        if (dim == 0) return bad("dim is 0");
        if (!d_a || !d_b || !d_out) return bad("null array");
        if (a_stride < dim || b_stride < dim || out_stride < n) return bad("a row stride is less than the row");
        if (!aligned_to(d_a_scale, 4) || !aligned_to(d_b_scale, 4) || !aligned_to(d_out, dtype_bytes(out_dtype)))
            return bad("an array is not aligned to its elements");
        if (dim > DIM_MAX) return set_error(TRAG_UNSUPPORTED, std::string(who) + ": a sum of more than 131071 products can pass 32 bits");
        // (a grid is at most 2^32 threads: 2^24 tiles of 128 x 128)
        if ((((uint64_t)m + 127) / 128) * (((uint64_t)n + 127) / 128) >= (1ull << 24))
            return set_error(TRAG_UNSUPPORTED, std::string(who) + ": the product has 2^24 tiles of 128 x 128 or more: split it");
        OpDevice on(who, hip_stream, {d_a, d_a_scale, d_b, d_b_scale, d_out});
        if (on.status != TRAG_OK) return on.status;
        const MmArgs p{d_a, d_b, d_a_scale, d_b_scale, d_out, a_stride, b_stride, out_stride, m, n, dim};
        const hipStream_t st = (hipStream_t)hip_stream;
        if (out_dtype == TRAG_F32) launch_mm<F32>(p, st);
        else if (out_dtype == TRAG_F16) launch_mm<F16>(p, st);
        else launch_mm<BF16>(p, st);
        return op_launched(who);
    });
}
