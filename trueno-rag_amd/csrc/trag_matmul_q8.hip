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

// The end of a row that is not a multiple of the step: a chunk of 16 bytes that would reach over the end is
// read at dim - 16 instead, in both operands alike (a sum does not mind the order of its terms), and in a the
// bytes that an earlier chunk has already brought are zero. b is never masked, and nothing is read outside a row.
__device__ __forceinline__ uint32_t chunk_at(uint32_t k, uint32_t dim) { return min(k, dim - 16u); }

__device__ __forceinline__ v4i load16(const int8_t* p) { return *reinterpret_cast<const v4i_any*>(p); }

// zeros the bytes of a chunk of a that stand for terms before k (the chunk was read at chunk_at(k, dim))
__device__ __forceinline__ v4i mask_chunk(v4i v, uint32_t k, uint32_t dim) {
    if (k + 16u <= dim) return v;
    const uint32_t cut = min(k - (dim - 16u), 16u);
#pragma unroll
    for (uint32_t w = 0; w < 4u; ++w) {
        const uint32_t c = cut > 4u * w ? min(cut - 4u * w, 4u) : 0u;
        v[w] = c == 4u ? 0 : (int)((uint32_t)v[w] & (0xFFFFFFFFu << (8u * c)));
    }
    return v;
}

// Rows shorter than a chunk, byte by byte, zeros behind the end.
__device__ __forceinline__ v4i load_short(const int8_t* row, uint32_t k, uint32_t dim) {
    v4i r = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 16u; ++i)
        if (k + i < dim) r[i >> 2] |= (int)((uint32_t)(uint8_t)row[k + i] << (8u * (i & 3u)));
    return r;
}

__device__ __forceinline__ float scaled(int acc, float sa, float sb) { return (float)acc * sa * sb; }

// Where the workgroups of a product go: consecutive workgroups land on different dies, each with a cache of its
// own, so each die gets a run of tiles, walked in columns of GM tiles of a: the tiles a die works on at one
// time then share rows of both operands.
struct TilePos {
    uint32_t m, n;
    bool there;
};
__device__ __forceinline__ TilePos tile_of(uint32_t b, uint32_t m_tiles, uint32_t n_tiles) {
    constexpr uint32_t GM = 4;
    const uint32_t tiles = m_tiles * n_tiles, per = (tiles + 7u) / 8u;
    const uint32_t t = (b & 7u) * per + (b >> 3);
    if ((b >> 3) >= per || t >= tiles) return {0, 0, false};
    const uint32_t g = t / (GM * n_tiles), g0 = g * GM, rows = min(GM, m_tiles - g0), in = t - g * GM * n_tiles;
    return {g0 + in % rows, in / rows, true};
}

// ---- rows shorter than a chunk, or 2^24 bytes and more apart, straight into matrix fragments: a wave takes 16 MT rows of a
// and 16 NT rows of b; lane l holds 16 bytes of row l % 16 from k = 16 (l / 16) on, so a wave-instruction reads 64 consecutive
// bytes of each of 16 rows. Nothing goes through LDS but the joining of partial sums where WK waves share one tile's terms. U:
// 64-byte steps whose loads are in flight together; the next U are asked for before the current ones are used. WN: tiles side
// by side in one workgroup.
template <typename T, int MT, int NT, int WK, int WN, int U, bool SHORT>
__global__ void __launch_bounds__(64 * WK * WN) mm_direct_kernel(const MmArgs p) {
    typedef typename T::elem E;
    constexpr int FR = MT * NT * 4;   // sums of a lane
    constexpr int PARTS = WK > 1 ? WK / 2 : 1;
    __shared__ int part[PARTS][WK > 1 ? WN * FR * 64 : 1];
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wid = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t wk = wid % WK, wn = wid / WK;
    const uint32_t m_tiles = (p.m + 16u * MT - 1u) / (16u * MT);
    const TilePos at = tile_of(blockIdx.x, m_tiles, (uint32_t)(((uint64_t)p.n + 16u * NT * WN - 1u) / (16u * NT * WN)));
    if (!at.there) return;   // (the whole workgroup)
    const uint32_t m0 = at.m * (16u * MT);
    const uint64_t n0 = ((uint64_t)at.n * WN + wn) * (16u * NT);
    const uint32_t r16 = lane & 15u, kq = (lane >> 4) * 16u;
    const uint32_t steps = (p.dim + 63u) / 64u;
    const uint32_t per = (steps + WK - 1u) / WK;
    const uint32_t s0 = min(wk * per, steps), s1 = min(s0 + per, steps);
    const int8_t *ar[MT], *br[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) ar[i] = p.a + (uint64_t)min(m0 + (uint32_t)i * 16u + r16, p.m - 1u) * p.lda;
#pragma unroll
    for (int j = 0; j < NT; ++j) br[j] = p.b + min(n0 + (uint32_t)j * 16u + r16, (uint64_t)p.n - 1u) * p.ldb;
    v4i acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = v4i{0, 0, 0, 0};
    v4i fa[2][U][MT], fb[2][U][NT];
    auto fetch = [&](int buf, uint32_t s) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + (uint32_t)u >= s1) continue;   // (wave-uniform)
            const uint32_t k = (s + (uint32_t)u) * 64u + kq;
#pragma unroll
            for (int j = 0; j < NT; ++j) fb[buf][u][j] = SHORT ? load_short(br[j], k, p.dim) : load16(br[j] + chunk_at(k, p.dim));
#pragma unroll
            for (int i = 0; i < MT; ++i) fa[buf][u][i] = SHORT ? load_short(ar[i], k, p.dim) : load16(ar[i] + chunk_at(k, p.dim));
        }
    };
    auto multiply = [&](int buf, uint32_t s) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + (uint32_t)u >= s1) continue;
            const bool last = !SHORT && (s + (uint32_t)u + 1u) * 64u > p.dim;
            const uint32_t k = (s + (uint32_t)u) * 64u + kq;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const v4i x = last ? mask_chunk(fa[buf][u][i], k, p.dim) : fa[buf][u][i];
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, fb[buf][u][j], acc[i][j], 0, 0, 0);
            }
        }
    };
    fetch(0, s0);
    for (uint32_t s = s0; s < s1; s += 2u * U) {
        fetch(1, s + U);
        multiply(0, s);
        fetch(0, s + 2u * U);
        multiply(1, s + U);
    }
    // the waves' sums joined two by two: half of those left hand theirs over, half add
    if constexpr (WK > 1) {
#pragma unroll
        for (int half = WK / 2; half >= 1; half /= 2) {
            if (wk >= (uint32_t)half && wk < 2u * half) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) part[wk - half][(wn * FR + (uint32_t)((i * NT + j) * 4 + r)) * 64u + lane] = acc[i][j][r];
            }
            __syncthreads();
            if (wk < (uint32_t)half) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i][j][r] += part[wk][(wn * FR + (uint32_t)((i * NT + j) * 4 + r)) * 64u + lane];
            }
            if (half > 1) __syncthreads();
        }
        if (wk > 0) return;
    }
    // lane l holds column l % 16 of rows 4 (l / 16) .. + 3
    E* const out = reinterpret_cast<E*>(p.out);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const uint64_t col = n0 + (uint32_t)j * 16u + r16;
        if (col >= p.n) continue;
        const float sb = p.sb ? p.sb[col] : 1.0f;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t row = m0 + (uint32_t)i * 16u + (lane >> 4) * 4u + (uint32_t)r;
                if (row < p.m) *(out + (uint64_t)row * p.ldo + col) = T::round(scaled(acc[i][j][r], p.sa ? p.sa[row] : 1.0f, sb));
            }
    }
}

// ---- tiles through LDS: WM x WN waves of (16 MT) x (16 NT) sums each, 128 bytes of every row a step. Bound by the
// matrix cores where there are tiles enough. LDS rows are 128 bytes without padding; chunk c of row r stands at
// slot c ^ (r / 2 % 8), so that the 16 rows of a fragment read fall on different banks.
// DMA: rows start on 16 bytes. Both operands go from memory straight into LDS (16 bytes a lane, no registers on the
// way; the permutation is applied to the addresses that the lanes fetch), ST stages deep. Otherwise the same through
// registers, two stages.
// KG: groups of waves that share a tile's terms, each with stages of its own, where there are few tiles.
// What bounds it (4096 x 16384 x 4096, 237 to 245 us from card to card, 2.3 POP/s; 8192 x 8192 x 8192 437 us, 2.5): the matrix cores
// at the 1.9 to 2.0 GHz that they hold under this load are busy 58 % of the cycles, LDS 25 %, bank conflicts 1.4 % among them;
// reading fragments ahead of the multiplications (128 x 128 tiles 355 -> 303 us) and moving the transfers within a step do not
// change the largest tile's time. A plain large 8-bit library product takes 288 and 527 us for the two.
// Where the terms are few or the tiles do not fill the CUs the time is 1.6 to 2.3 times that of the traffic or of the matrix cores:
// 4096 x 16384 x 384 bf16 65 us of 27, f32 93 of 53, 1000 x 50000 x 384 f32 70 of 42, 315 x 7024 x 7936 39 of 17. A 256 x 256
// tile of 384 terms is three steps and 4.9 us of filling stages and epilogue with nothing beside it on the CU; 165 tiles of 128 x 128 are
// fewer than the CUs.
template <typename T, int WM, int WN, int MT, int NT, int KG, int ST, bool DMA>
__global__ void __launch_bounds__(64 * WM * WN * KG, 2) mm_tile_kernel(const MmArgs p) {
    typedef typename T::elem E;
    constexpr int NW = WM * WN;
    constexpr uint32_t BM = 16u * MT * WM, BN = 16u * NT * WN;
    constexpr uint32_t STAGE = (BM + BN) * 128u;
    constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW;      // pieces (8 rows, 1 KB) of each operand a wave brings a step
    static_assert(PA * NW * 8 == (int)BM && PB * NW * 8 == (int)BN, "whole pieces");
    static_assert(DMA || ST == 2, "through registers: two stages");
    // (through registers the largest tile has none left for a second set of fragments: 110 of them would spill, 414 us
    // instead of 157 for 4096 x 8192 x 4001)
    constexpr bool AHEAD = DMA || MT * NT <= 16;
    constexpr uint32_t PER = 16u / sizeof(E);              // elements of 16 bytes
    constexpr uint32_t RUN = 16u * NT, LDO = RUN + PER;    // a row of a wave's piece of the epilogue
    static_assert(NW * 16u * LDO * sizeof(E) <= ST * STAGE, "the epilogue's pieces fit the stages");
    constexpr int FR = MT * NT * 4;                        // sums of a lane
    static_assert(KG == 1 || KG / 2 * NW * FR * 256 <= (int)(KG * ST * STAGE), "the sums that are handed over fit the stages");
    __shared__ __attribute__((aligned(1024))) int8_t all[KG * ST * STAGE];
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t kg = wave / NW, wid = wave % NW;
    int8_t* const lds = all + kg * (ST * STAGE);           // (each group of waves has stages of its own)
    const uint32_t wm = wid / WN, wn = wid % WN;
    const TilePos at = tile_of(blockIdx.x, (p.m + BM - 1u) / BM, (uint32_t)(((uint64_t)p.n + BN - 1u) / BN));
    if (!at.there) return;
    const uint32_t m0 = at.m * BM, n0 = at.n * BN;
    // the terms are dealt out to the groups in runs; every group passes the same barriers, with or without a step to do
    const uint32_t total = (p.dim + 127u) / 128u, rounds = (total + KG - 1u) / KG;
    const uint32_t first = min(kg * rounds, total), steps = min(rounds, total - first);
    uint32_t oa[PA], ob[PB];                               // byte offsets of a lane's chunks from the tile's first row
    const uint32_t c8 = (lane & 7u);
#pragma unroll
    for (int i = 0; i < PA; ++i) {
        const uint32_t row = (wid * PA + (uint32_t)i) * 8u + (lane >> 3);
        oa[i] = (min(m0 + row, p.m - 1u) - m0) * (uint32_t)p.lda + (c8 ^ ((row >> 1) & 7u)) * 16u;
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) {
        const uint32_t row = (wid * PB + (uint32_t)i) * 8u + (lane >> 3);
        ob[i] = (min(n0 + row, p.n - 1u) - n0) * (uint32_t)p.ldb + (c8 ^ ((row >> 1) & 7u)) * 16u;
    }
    const int8_t* const abase = p.a + (uint64_t)m0 * p.lda;
    const int8_t* const bbase = p.b + (uint64_t)n0 * p.ldb;
    // bytes by which a chunk of the last step is moved back to end at the row's end (or 0)
    auto back = [&](uint32_t step, uint32_t first_row, int i) __attribute__((always_inline)) {
        const uint32_t row = first_row + (uint32_t)i * 8u + (lane >> 3);
        const uint32_t k = step * 128u + (c8 ^ ((row >> 1) & 7u)) * 16u;
        return k - chunk_at(k, p.dim);
    };
    typedef __attribute__((address_space(3))) int8_t* lds_ptr;
    v4i ra[DMA ? 1 : PA], rb[DMA ? 1 : PB];
    auto transfer = [&](uint32_t slot, uint32_t step) __attribute__((always_inline)) {
        const int8_t* const sa = abase + (uint64_t)step * 128u;
        const int8_t* const sb = bbase + (uint64_t)step * 128u;
        const bool whole = (step + 1u) * 128u <= p.dim;
        if constexpr (DMA) {
#if defined(__HIP_DEVICE_COMPILE__)
            const uint32_t to = (uint32_t)(uintptr_t)(lds_ptr)lds + slot * STAGE;
            const uint32_t ta = to + wid * (PA * 1024u), tb = to + BM * 128u + wid * (PB * 1024u);
            if (whole) {
#pragma unroll
                for (int i = 0; i < PA; ++i) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(ta + (uint32_t)i * 1024u), "v"(oa[i]), "s"(sa) : "memory");
#pragma unroll
                for (int i = 0; i < PB; ++i) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(tb + (uint32_t)i * 1024u), "v"(ob[i]), "s"(sb) : "memory");
            } else {   // (dim is a multiple of 16 here: a chunk is whole, or moved back to the row's last one)
#pragma unroll
                for (int i = 0; i < PA; ++i) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(ta + (uint32_t)i * 1024u), "v"(oa[i] - back(step, wid * PA * 8u, i)), "s"(sa) : "memory");
#pragma unroll
                for (int i = 0; i < PB; ++i) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(tb + (uint32_t)i * 1024u), "v"(ob[i] - back(step, wid * PB * 8u, i)), "s"(sb) : "memory");
            }
#endif
        } else {
#pragma unroll
            for (int i = 0; i < PA; ++i) ra[i] = load16(sa + oa[i] - (whole ? 0u : back(step, wid * PA * 8u, i)));
#pragma unroll
            for (int i = 0; i < PB; ++i) rb[i] = load16(sb + ob[i] - (whole ? 0u : back(step, wid * PB * 8u, i)));
        }
    };
    auto piece = [&](uint32_t slot, uint32_t step, int x) __attribute__((always_inline)) {   // one instruction of a whole step's transfer
#if defined(__HIP_DEVICE_COMPILE__)
        const uint32_t to = (uint32_t)(uintptr_t)(lds_ptr)lds + slot * STAGE;
        if (x < PA)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to + (wid * PA + (uint32_t)x) * 1024u), "v"(oa[x < PA ? x : 0]), "s"(abase + (uint64_t)step * 128u) : "memory");
        else
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to + BM * 128u + (wid * PB + (uint32_t)(x - PA)) * 1024u), "v"(ob[x < PA ? 0 : x - PA]), "s"(bbase + (uint64_t)step * 128u) : "memory");
#endif
    };
    auto put = [&](uint32_t slot) __attribute__((always_inline)) {   // (through registers: what transfer() brought, into LDS)
        if constexpr (!DMA) {
            int8_t* const to = lds + slot * STAGE + lane * 16u;
#pragma unroll
            for (int i = 0; i < PA; ++i) *reinterpret_cast<v4i*>(to + (wid * PA + (uint32_t)i) * 1024u) = ra[i];
#pragma unroll
            for (int i = 0; i < PB; ++i) *reinterpret_cast<v4i*>(to + BM * 128u + (wid * PB + (uint32_t)i) * 1024u) = rb[i];
        }
    };
    v4i acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = v4i{0, 0, 0, 0};
    const uint32_t r16 = lane & 15u, q = lane >> 4;
    const uint32_t sw = (r16 >> 1) & 7u;
    const uint32_t fra = (wm * (16u * MT) + r16) * 128u, frb = BM * 128u + (wn * (16u * NT) + r16) * 128u;
    // a half of a step (64 bytes of every row) into fragments
    auto frags = [&](uint32_t slot, uint32_t h, v4i (&xa)[MT], v4i (&xb)[NT]) __attribute__((always_inline)) {
        const int8_t* const S = lds + slot * STAGE;
        const uint32_t c = ((h * 4u + q) ^ sw) * 16u;
#pragma unroll
        for (int j = 0; j < NT; ++j) xb[j] = *reinterpret_cast<const v4i*>(S + frb + j * 2048 + c);
#pragma unroll
        for (int i = 0; i < MT; ++i) xa[i] = *reinterpret_cast<const v4i*>(S + fra + i * 2048 + c);
    };
    auto mfma_row = [&](int i, const v4i (&xa)[MT], const v4i (&xb)[NT]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xb[j], xa[i], acc[i][j], 0, 0, 0);
    };
    auto multiply_last = [&](uint32_t slot, uint32_t step) __attribute__((always_inline)) {   // a step that is not whole
#pragma unroll 1
        for (uint32_t h = 0; h < 2u; ++h) {
            const uint32_t k = step * 128u + h * 64u;
            if (k >= p.dim) break;
            v4i xa[MT], xb[NT];
            frags(slot, h, xa, xb);
#pragma unroll
            for (int i = 0; i < MT; ++i) xa[i] = mask_chunk(xa[i], k + q * 16u, p.dim);
#pragma unroll
            for (int i = 0; i < MT; ++i) mfma_row(i, xa, xb);
        }
    };
    // The loop meets once a step, in its middle: the second half's fragments are read while the first half multiplies; then the
    // waves meet -- this step's stage has been read, the next one's has landed --, and while the second half multiplies the
    // stage is filled again and the next step's first fragments are read. The matrix cores wait for neither.
    const uint32_t whole = min(steps, p.dim / 128u - min(first, p.dim / 128u));   // steps without an end of the rows
    v4i fa0[MT], fb0[NT], fa1[MT], fb1[NT];
    if constexpr (DMA) {
#pragma unroll
        for (uint32_t s = 0; s < (uint32_t)ST; ++s)
            if (s < steps) transfer(s, first + s);
        if (ST <= (int)steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 1) * (PA + PB)) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else {
        if (steps > 0) { transfer(0, first); put(0); }
        if (AHEAD && steps > 1) { transfer(1, first + 1u); put(1); }
        if (AHEAD && steps > 2) transfer(0, first + 2u);
    }
    __syncthreads();
    uint32_t slot = 0, s = 0;
    if constexpr (!AHEAD) {
        for (; s < whole; ++s) {   // (the next step's loads are in flight while this one multiplies)
            if (s + 1u < steps) transfer(0, first + s + 1u);
#pragma unroll
            for (uint32_t h = 0; h < 2u; ++h) {
                frags(slot, h, fa0, fb0);
#pragma unroll
                for (int i = 0; i < MT; ++i) mfma_row(i, fa0, fb0);
            }
            slot ^= 1u;
            if (s + 1u < steps) put(slot);
            __syncthreads();
        }
    }
    if constexpr (AHEAD) frags(0, 0, fa0, fb0);
    for (; AHEAD && s < whole; ++s) {
        const uint32_t next = slot + 1u == (uint32_t)ST ? 0u : slot + 1u;
        frags(slot, 1, fa1, fb1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < MT; ++i) mfma_row(i, fa0, fb0);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (DMA) {   // the next step's transfers are in; those of up to ST - 2 more may be on their way
            if (ST == 2 || s + (uint32_t)ST <= steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 2) * (PA + PB)) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        __syncthreads();
        if constexpr (!DMA)
            if (s + 2u < steps) put(slot);
        frags(next, 0, fa0, fb0);   // (behind the last step: of no use, of no harm)
        __builtin_amdgcn_sched_barrier(0);
        // (a transfer behind every few multiplications; two, four or all of them together take the same time)
        const bool more = s + (uint32_t)ST < whole;
        if constexpr (DMA) {
            if (!more && s + (uint32_t)ST < steps) transfer(slot, first + s + (uint32_t)ST);
        } else {
            if (s + 3u < steps) transfer(0, first + s + 3u);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if constexpr (DMA) {
                if (more) {
#pragma unroll
                    for (int x = 0; x < PA + PB; ++x)
                        if (x * MT / (PA + PB) == i) piece(slot, first + s + (uint32_t)ST, x);
                }
            }
            mfma_row(i, fa1, fb1);
            if constexpr (DMA) __builtin_amdgcn_sched_barrier(0);
        }
        slot = next;
    }
    if (whole < steps) multiply_last(slot, first + whole);
    for (; s < rounds; ++s) __syncthreads();   // (a group with fewer steps passes the others' meetings)
    __syncthreads();
    // the groups' sums joined two by two: half of those left hand theirs over, half add
    if constexpr (KG > 1) {
        int* const part = reinterpret_cast<int*>(all);
#pragma unroll
        for (uint32_t half = KG / 2; half >= 1u; half /= 2u) {
            if (kg >= half && kg < 2u * half) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        *reinterpret_cast<v4i*>(part + ((((kg - half) * NW + wid) * (MT * NT) + (uint32_t)(i * NT + j)) * 64u + lane) * 4u) = acc[i][j];
            }
            __syncthreads();
            if (kg < half) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        acc[i][j] += *reinterpret_cast<const v4i*>(part + (((kg * NW + wid) * (MT * NT) + (uint32_t)(i * NT + j)) * 64u + lane) * 4u);
            }
            __syncthreads();
        }
        if (kg > 0) return;
    }
    // b's rows came first in the multiplications: lane l holds row l % 16 and columns 4 (l / 16) .. + 3 of every 16 x 16 block,
    // which go side by side into a piece of LDS of the wave's own, 16 rows at a time; read back along the rows, a store
    // covers whole runs of a row. (A wave's LDS accesses are served in order.)
    E* const out = reinterpret_cast<E*>(p.out);
    E* const block = reinterpret_cast<E*>(all) + wid * (16u * LDO);
    typedef E evec __attribute__((ext_vector_type(16 / sizeof(E)), aligned(sizeof(E))));
    typedef E four __attribute__((ext_vector_type(4)));
    typedef float scale4 __attribute__((ext_vector_type(4), aligned(4)));
    const uint32_t col0 = n0 + wn * RUN, row00 = m0 + wm * (16u * MT);
    scale4 sb[NT];
    float sa[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const uint32_t col = col0 + (uint32_t)j * 16u + q * 4u;
        sb[j] = scale4{1.0f, 1.0f, 1.0f, 1.0f};
        if (p.sb) {
            if (col + 4u <= p.n) sb[j] = *reinterpret_cast<const scale4*>(p.sb + col);
            else
#pragma unroll
                for (uint32_t r = 0; r < 4u; ++r)
                    if (col + r < p.n) sb[j][r] = p.sb[col + r];
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) sa[i] = p.sa ? p.sa[min(row00 + (uint32_t)i * 16u + r16, p.m - 1u)] : 1.0f;
    constexpr uint32_t LPR = RUN / PER;                           // lanes a row
    constexpr uint32_t RPI = 64u / LPR < 16u ? 64u / LPR : 16u;   // rows a wave-instruction
    const uint32_t c = (lane % LPR) * PER;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            four v;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = T::round(scaled(acc[i][j][r], sa[i], sb[j][r]));
            *reinterpret_cast<four*>(block + r16 * LDO + (uint32_t)j * 16u + q * 4u) = v;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        evec v[16u / RPI];
#pragma unroll
        for (uint32_t r = 0; r < 16u / RPI; ++r) v[r] = *reinterpret_cast<const evec*>(block + min(r * RPI + lane / LPR, 15u) * LDO + c);
#pragma unroll
        for (uint32_t r = 0; r < 16u / RPI; ++r) {
            const uint32_t lr = r * RPI + lane / LPR, row = row00 + (uint32_t)i * 16u + lr;
            if (lr < 16u && row < p.m) {
                E* const to = out + (uint64_t)row * p.ldo + col0 + c;
                if (col0 + c + PER <= p.n) *reinterpret_cast<evec*>(to) = v[r];
                else
#pragma unroll
                    for (uint32_t x = 0; x < PER; ++x)
                        if (col0 + c + x < p.n) to[x] = v[r][x];
            }
        }
    }
}

uint32_t grid8(uint64_t tiles) { return (uint32_t)((tiles + 7u) / 8u * 8u); }   // (a run of tiles for each of 8 dies)

// (A grid's threads are counted in 32 bits: a product of more tiles goes out in several launches.)
template <typename T, int MT, int NT, int WK, int WN, int U, bool SHORT = false>
void launch_direct(const MmArgs& p, hipStream_t st) {
    constexpr uint32_t BM = 16u * MT, BN = 16u * NT * WN, most = 0xFFFFFFFFu / (64u * WK * WN) - 8u;
    const uint32_t mt = (p.m + BM - 1u) / BM, nt = (uint32_t)(((uint64_t)p.n + BN - 1u) / BN);
    const uint32_t n_run = nt < most ? nt : most, m_run = mt < most / n_run ? mt : most / n_run;
    for (uint32_t m0 = 0; m0 < mt; m0 += m_run)
        for (uint32_t n0 = 0; n0 < nt; n0 += n_run) {
            MmArgs q = p;
            q.m = (mt - m0 <= m_run ? p.m - m0 * BM : m_run * BM);
            q.n = (nt - n0 <= n_run ? p.n - n0 * BN : n_run * BN);
            q.a = p.a + (uint64_t)m0 * BM * p.lda;
            q.b = p.b + (uint64_t)n0 * BN * p.ldb;
            if (p.sa) q.sa = p.sa + m0 * BM;
            if (p.sb) q.sb = p.sb + n0 * BN;
            q.out = reinterpret_cast<typename T::elem*>(p.out) + (uint64_t)m0 * BM * p.ldo + n0 * BN;
            const uint64_t tiles = (uint64_t)((q.m + BM - 1u) / BM) * (((uint64_t)q.n + BN - 1u) / BN);
            hipLaunchKernelGGL((mm_direct_kernel<T, MT, NT, WK, WN, U, SHORT>), dim3(grid8(tiles)), dim3(64 * WK * WN), 0, st, q);
        }
}

template <typename T, int WM, int WN, int MT, int NT, int KG, int ST, bool DMA>
void launch_tile(const MmArgs& p, hipStream_t st) {
    constexpr uint32_t BM = 16u * MT * WM, BN = 16u * NT * WN;
    const uint64_t tiles = (uint64_t)((p.m + BM - 1u) / BM) * (((uint64_t)p.n + BN - 1u) / BN);
    hipLaunchKernelGGL((mm_tile_kernel<T, WM, WN, MT, NT, KG, ST, DMA>), dim3(grid8(tiles)), dim3(64 * WM * WN * KG), 0, st, p);
}

// Transfers straight into LDS: whole 16-byte chunks at addresses that are multiples of 16.
bool dma_fits(const MmArgs& p) {
    return p.dim % 16u == 0 && p.lda % 16u == 0 && p.ldb % 16u == 0 && aligned_to(p.a, 16) && aligned_to(p.b, 16);
}

// Which tile. Every form gives the same bits, so the choice is one of time alone: the one with the least
//   max(rounds (fix + per * steps a group of waves does), operands and output / 6 TB/s + what tiles read again / 16 TB/s),
// rounds = tiles over what 256 CUs work on at once; `per`, the time of a 128-byte step, grows from `lo` to `hi` as the CUs fill
// up (12 TB/s for rows at any byte). The constants are fitted, form by form, to the times of 1900 products of random sizes
// (1 to 4096 by 64 to 1M by 32 to 8192); over 1000 others the choice takes 1.8 % longer than the best form on average, 11 % in
// the worst twentieth (against the best form, not against what the traffic allows). Some of the times (us of the kernel among others of its kind; bf16 output; aligned rows, m x n x dim):
//   16 x 4096 x 4096   16 x 16 tiles in 8 groups of waves  6.3    16 x 32 in 4  6.4    16 x 64 in 4  7.5    in 1  16.6
//   8 x 2048 x 8192    16 x 16 in 8   6.4    16 x 32 in 4   8.2    16 x 64 in 4  10.5    in 1  30.3
//   100 x 1000 x 4096  16 x 32 in 4   6.2    16 x 64 in 4   7.4    32 x 64 in 4   8.3    16 x 16 in 8   8.4
//   256 x 4096 x 4096  64 x 64 in 2  10.6    32 x 64 in 4  11.3    in 1  18.0    128 x 128 in 2  20.1    in 1  24.0
//   1024 x 4096 x 4096 128 x 128 in 2  22.7    64 x 128  25.0    128 x 128 in 1  25.9    64 x 64 in 1  28.7    256 x 256  44.5
//   4096 x 16384 x 4096  256 x 256  235    128 x 128 in 1  290
//   1 x 1M x 384  16 x 64 in 1  66    64 x 1M x 384  64 x 128  102, 64 x 64  108    128 x 1M x 384  128 x 128  136, 64 x 64  180
// and for rows at any byte (through registers):
//   15 x 2154 x 7715  16 x 16 in 8  9.5, 16 x 32 in 4  12.8, 32 x 64 in 4  21.9    37 x 50021 x 777  64 x 128  12.2, 64 x 64  13.5
//   512 x 4096 x 4001  64 x 64  22.6, 64 x 128  23.0, 128 x 128  28.8    4096 x 8192 x 4001  256 x 256  150, 128 x 128  189
enum TileForm { T16x16G8, T16x32G4, T16, T16G4, T32, T32G4, T64, T64G2, T64x128, T128, T128G2, T256, N_FORMS };
struct FormCost {
    uint16_t bm, bn, groups, threads;
    uint16_t held;             // workgroups a CU works on at once (0: this form is not built)
    float fix, lo, hi;
};
constexpr FormCost DMA_COST[N_FORMS] = {
    {16, 16, 8, 512, 1, 0.83f, 0.26f, 0.66f},   {16, 32, 4, 512, 1, 0.98f, 0.24f, 0.51f},
    {16, 64, 1, 128, 5, 0.64f, 0.28f, 0.66f},   {16, 64, 4, 512, 1, 1.13f, 0.38f, 0.73f},   {32, 64, 1, 128, 6, 0.94f, 0.30f, 1.04f},
    {32, 64, 4, 512, 1, 1.36f, 0.48f, 0.89f},   {64, 64, 1, 256, 5, 1.04f, 0.31f, 1.20f},   {64, 64, 2, 512, 1, 1.53f, 0.34f, 0.60f},
    {64, 128, 1, 256, 3, 1.73f, 0.43f, 1.15f},  {128, 128, 1, 256, 2, 2.60f, 0.55f, 1.14f},
    {128, 128, 2, 512, 1, 3.12f, 0.92f, 1.42f}, {256, 256, 1, 512, 1, 4.93f, 1.21f, 1.78f}};
constexpr FormCost ANY_COST[N_FORMS] = {
    {16, 16, 8, 512, 1, 0.38f, 0.70f, 0.72f},   {16, 32, 4, 512, 1, 0.35f, 0.62f, 0.51f},
    {16, 64, 1, 128, 8, 0.91f, 0.34f, 1.70f},   {16, 64, 4, 512, 0, 0.0f, 0.0f, 0.0f},      {32, 64, 1, 128, 6, 1.22f, 0.36f, 1.62f},
    {32, 64, 4, 512, 1, 1.23f, 0.86f, 1.43f},   {64, 64, 1, 256, 5, 1.54f, 0.36f, 1.85f},   {64, 64, 2, 512, 0, 0.0f, 0.0f, 0.0f},
    {64, 128, 1, 256, 3, 2.18f, 0.53f, 1.73f},  {128, 128, 1, 256, 2, 3.07f, 0.81f, 1.65f},
    {128, 128, 2, 512, 0, 0.0f, 0.0f, 0.0f},    {256, 256, 1, 512, 1, 5.20f, 1.86f, 2.40f}};

int choose_form(const MmArgs& p, bool dma, uint32_t out_bytes) {
    constexpr double CUS = 256.0;
    const double steps = (double)((p.dim + 127u) / 128u);
    const double once = ((double)p.m + (double)p.n) * p.dim;
    int best = T256;
    double least = 1e300;
    for (int f = 0; f < N_FORMS; ++f) {
        const FormCost& c = dma ? DMA_COST[f] : ANY_COST[f];
        if (!c.held) continue;
        const double tiles = (double)((p.m + c.bm - 1u) / c.bm) * (double)(((uint64_t)p.n + c.bn - 1u) / c.bn);
        if ((tiles + 8.0) * c.threads >= 4294967296.0) continue;   // (a grid's threads are counted in 32 bits)
        const double at_once = CUS * c.held, full = tiles < at_once ? tiles / at_once : 1.0;
        const double rounds = __builtin_ceil(tiles / at_once);
        const double busy = rounds * (c.fix + (c.lo + (c.hi - c.lo) * full) * __builtin_ceil(steps / c.groups));
        const double again = tiles * (c.bm + c.bn) * (double)p.dim - once;
        const double moved = (once + (double)p.m * p.n * out_bytes) / 6.0e6 + (again > 0.0 ? again : 0.0) / (dma ? 16.0e6 : 12.0e6);
        const double t = busy > moved ? busy : moved;
        if (t < least) {
            least = t;
            best = f;
        }
    }
    return best;
}

template <typename T>
void launch_mm(const MmArgs& p, hipStream_t st) {
    if (p.dim < 16u) return launch_direct<T, 1, 8, 1, 4, 1, true>(p, st);
    // (the tiles' offsets from their first row are 32 bits, over 255 rows at most)
    if (p.lda >= (1u << 24) || p.ldb >= (1u << 24)) return launch_direct<T, 1, 1, 8, 1, 4>(p, st);
    const bool dma = dma_fits(p);
    const int form = choose_form(p, dma, sizeof(typename T::elem));
    if (dma) {
        switch (form) {
            case T16x16G8: return launch_tile<T, 1, 1, 1, 1, 8, 4, true>(p, st);
            case T16x32G4: return launch_tile<T, 1, 2, 1, 1, 4, 4, true>(p, st);
            case T16: return launch_tile<T, 1, 2, 1, 2, 1, 2, true>(p, st);
            case T16G4: return launch_tile<T, 1, 2, 1, 2, 4, 3, true>(p, st);
            case T32: return launch_tile<T, 1, 2, 2, 2, 1, 2, true>(p, st);
            case T32G4: return launch_tile<T, 1, 2, 2, 2, 4, 3, true>(p, st);
            case T64: return launch_tile<T, 2, 2, 2, 2, 1, 2, true>(p, st);
            case T64G2: return launch_tile<T, 2, 2, 2, 2, 2, 4, true>(p, st);
            case T64x128: return launch_tile<T, 2, 2, 2, 4, 1, 2, true>(p, st);
            case T128: return launch_tile<T, 2, 2, 4, 4, 1, 2, true>(p, st);
            case T128G2: return launch_tile<T, 2, 2, 4, 4, 2, 2, true>(p, st);
            default: return launch_tile<T, 4, 2, 4, 8, 1, 2, true>(p, st);
        }
    }
    switch (form) {
        case T16x16G8: return launch_tile<T, 1, 1, 1, 1, 8, 2, false>(p, st);
        case T16x32G4: return launch_tile<T, 1, 2, 1, 1, 4, 2, false>(p, st);
        case T16: return launch_tile<T, 1, 2, 1, 2, 1, 2, false>(p, st);
        case T32: return launch_tile<T, 1, 2, 2, 2, 1, 2, false>(p, st);
        case T32G4: return launch_tile<T, 1, 2, 2, 2, 4, 2, false>(p, st);
        case T64: return launch_tile<T, 2, 2, 2, 2, 1, 2, false>(p, st);
        case T64x128: return launch_tile<T, 2, 2, 2, 4, 1, 2, false>(p, st);
        case T128: return launch_tile<T, 2, 2, 4, 4, 1, 2, false>(p, st);
        default: return launch_tile<T, 4, 2, 4, 8, 1, 2, false>(p, st);
    }
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
        // (a grid's threads are counted in 32 bits)
        if ((((uint64_t)m + 127) / 128) * (((uint64_t)n + 127) / 128) >= (1ull << 22))
            return set_error(TRAG_UNSUPPORTED, std::string(who) + ": the product has 2^22 tiles of 128 x 128 or more: split it");
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
