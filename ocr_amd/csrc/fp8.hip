// 8-bit floating point products with a scale for each block of 128 (no counterpart in the reference, which computes in
// float32).
//
//   quantise:  the values of a block (1 x 128, or 128 x 128 of a weight matrix) are divided by a power of two 2^e, the
//              least with amax <= 448 * 2^e (448 is the largest e4m3 value), and rounded to e4m3 (nearest, ties to even):
//              the division is exact, so the only rounding is that to four significant bits.
//   product:   C[m,n] = sum over blocks j of 2^(ea[m,j] + eb[n,j]) * sum over k in j of A[m,k] * B[n,k]  (+ bias[n])
//
// The scales are powers of two because a value times its scale is then a bfloat16 number, and the conversion instruction takes
// the scale itself: the products of all blocks add up in ONE float32 accumulator, without a multiply-add of every accumulator
// by a float scale after each block.  A float scale would use the range of e4m3 better by less than a factor of 2, which a
// floating type does not need: the relative rounding error is 2^-4 at any magnitude.
//
// Sums are float32: the bytes times their scale are converted to bfloat16 on the way from LDS (exact: 4 significant bits) and
// multiplied by v_mfma_f32_16x16x32_bf16.  The 8-bit matrix instructions, at twice its rate, would not do: they add the
// products of a group of neighbouring values of k (at most 16) aligned to the largest of them and keep 13 bits below it
// (measured, with and without scales: a product 2^-14 of its neighbour's is lost, one 16 places further is not).  448 * 448 -
// 448 * 448 + 4 gave 0, and 3.8 % of a large product's bfloat16 results were other roundings than those of float32 sums.  The
// price: 8192^3 into bfloat16 takes 794 us instead of 440, 2048^3 23 instead of 15, 79872 x 256 x 512 25 as before.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "common.h"
#include "scale_window.h"

namespace ocrhip {

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

std::mutex g_lds_mutex;              // guards the once-per-device LDS opt-in of the kernels that need more than 64 KB

constexpr int kBlk = 128;            // values of k that share a scale
constexpr int kBias = 127;           // stored byte = exponent + 127 (255 is no exponent: the instruction takes it as NaN)

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const uint16_t* p) { return __uint_as_float((unsigned)*p << 16); }

// Stored exponent byte of a block whose largest finite magnitude is amax: amax = m * 2^x with 1 <= m < 2 fits 448 =
// 1.75 * 2^8 after a division by 2^(x-8) if m <= 1.75, else by 2^(x-7).  Subnormal amax: x is below -126 and the exponent
// is clamped at -127 anyway.  A block of zeros takes 2^0.
__device__ __forceinline__ unsigned scale_byte(float amax) {
    const unsigned u = __float_as_uint(amax);
    if (u == 0) return kBias;
    const int x = (int)(u >> 23) - 127;
    const int e = x - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return (unsigned)(max(e, -127) + kBias);
}

// 2^-(byte - 127): between 2^127 (byte 0, the clamped exponent) and 2^-120 (byte 247, the largest finite float's), a float
// for every byte that occurs
__device__ __forceinline__ float inverse_scale(unsigned byte) { return ldexpf(1.0f, kBias - (int)byte); }

// what counts for amax: infinities and NaN become NaN in e4m3 whatever the scale
__device__ __forceinline__ float finite_magnitude(float v) {
    const float a = fabsf(v);
    return a < INFINITY ? a : 0.0f;
}

__device__ __forceinline__ unsigned pack4_e4m3(float a, float b, float c, float d) {
    int r = 0;
    r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    return (unsigned)r;
}

// an infinity would saturate to the largest value in the conversion: make it a NaN first
__device__ __forceinline__ float no_infinity(float v) { return fabsf(v) == INFINITY ? __uint_as_float(0x7FC00000u) : v; }

// Vectors at the alignment of their elements: rows of odd length start anywhere, and global memory takes 16-byte accesses
// at any element.
typedef float floatx4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef int intx4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x8_any __attribute__((ext_vector_type(8), aligned(2)));

// NV (a multiple of 8) values x[k0 ..] of a row of K, zeros beyond
template <int NV>
__device__ __forceinline__ void load_run(const float* x, int64_t k0, int64_t K, float* v) {
    if (k0 + NV <= K) {
#pragma unroll
        for (int e = 0; e < NV; e += 4) {
            const floatx4 t = *reinterpret_cast<const floatx4_any*>(x + k0 + e);
            v[e] = t[0]; v[e + 1] = t[1]; v[e + 2] = t[2]; v[e + 3] = t[3];
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < NV; ++e) v[e] = k0 + e < K ? x[k0 + e] : 0.0f;
}
template <int NV>
__device__ __forceinline__ void load_run(const uint16_t* x, int64_t k0, int64_t K, float* v) {
    if (k0 + NV <= K) {
#pragma unroll
        for (int e = 0; e < NV; e += 8) {
            const intx4 t = *reinterpret_cast<const intx4_any*>(x + k0 + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[e + 2 * i] = __int_as_float(t[i] << 16);
                v[e + 2 * i + 1] = __int_as_float(t[i] & (int)0xFFFF0000);
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < NV; ++e) v[e] = k0 + e < K ? load_f32(x + k0 + e) : 0.0f;
}

// ---- quantise
//
// Bound by reading x and writing the bytes once (131072 x 512 bfloat16: 42 us, 4.75 TB/s; the transpose of 16384 x 6719
// float32: 110 us, 5 TB/s).  16 lanes hold a block of a row, 8 values each (one or two 16-byte loads,
// 8 bytes to store); the maximum crosses them by four exchanges.
constexpr int kRowsWg = 16;           // rows a workgroup of 256 threads works on at a time
constexpr int kBlocksWg = 4;          // column blocks it walks: their loads are in flight together

__device__ __forceinline__ float max16(float v) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

__device__ __forceinline__ uint64_t pack8_e4m3(const float* v, float inv) {
    float t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = no_infinity(v[e] * inv);
    return (uint64_t)pack4_e4m3(t[0], t[1], t[2], t[3]) | (uint64_t)pack4_e4m3(t[4], t[5], t[6], t[7]) << 32;
}

// one scale per row and 128 columns: 16 rows x 4 column blocks
template <class T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int64_t ld_x, int64_t rows, int64_t cols, uint8_t* __restrict__ q,
                                                            int64_t ld_q, uint8_t* __restrict__ scale, int64_t ld_s, unsigned chunks) {
    const int part = threadIdx.x & 15, sub = threadIdx.x >> 4;
    const int64_t row = (int64_t)(blockIdx.x / chunks) * kRowsWg + sub, kb0 = (int64_t)(blockIdx.x % chunks) * kBlocksWg;
    const int nkb = (int)min((int64_t)kBlocksWg, (cols + kBlk - 1) / kBlk - kb0);
    const bool there = row < rows;
    const T* p = x + (there ? row : 0) * ld_x;
    float v[kBlocksWg][8];
#pragma unroll
    for (int i = 0; i < kBlocksWg; ++i)
        if (i < nkb) load_run<8>(p, (kb0 + i) * kBlk + part * 8, cols, v[i]);
#pragma unroll
    for (int i = 0; i < kBlocksWg; ++i) {
        if (i >= nkb) break;
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_magnitude(v[i][e]));
        const unsigned byte = scale_byte(max16(amax));
        if (!there) continue;
        *reinterpret_cast<uint64_t*>(q + row * ld_q + (kb0 + i) * kBlk + part * 8) = pack8_e4m3(v[i], inverse_scale(byte));
        if (part == 0) scale[(kb0 + i) * ld_s + row] = (uint8_t)byte;
    }
}

// one scale per 128 rows x 128 columns: a workgroup holds the block in registers
template <class T>
__global__ __launch_bounds__(256) void quantize_block_kernel(const T* __restrict__ x, int64_t ld_x, int64_t rows, int64_t cols, uint8_t* __restrict__ q,
                                                             int64_t ld_q, uint8_t* __restrict__ scale, int64_t ld_s, unsigned col_blocks) {
    __shared__ float wave_max[4];
    const int part = threadIdx.x & 15, sub = threadIdx.x >> 4;
    const int64_t rb = blockIdx.x / col_blocks, cb = blockIdx.x % col_blocks;
    float v[kBlk / kRowsWg][8], amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kBlk / kRowsWg; ++i) {
        const int64_t row = rb * kBlk + i * kRowsWg + sub;
        if (row < rows) load_run<8>(x + row * ld_x, cb * kBlk + part * 8, cols, v[i]);
    }
#pragma unroll
    for (int i = 0; i < kBlk / kRowsWg; ++i) {
        if (rb * kBlk + i * kRowsWg + sub >= rows) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_magnitude(v[i][e]));
    }
    for (int o = 1; o < 64; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = amax;
    __syncthreads();
    const unsigned byte = scale_byte(fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3])));
    const float inv = inverse_scale(byte);
    if (threadIdx.x == 0) scale[cb * ld_s + rb] = (uint8_t)byte;
#pragma unroll
    for (int i = 0; i < kBlk / kRowsWg; ++i) {
        const int64_t row = rb * kBlk + i * kRowsWg + sub;
        if (row >= rows) break;
        *reinterpret_cast<uint64_t*>(q + row * ld_q + cb * kBlk + part * 8) = pack8_e4m3(v[i], inv);
    }
}

// The transpose of x: a workgroup reads 128 rows x WC columns (whole vectors along the rows), passes them through LDS (rows
// an odd number of floats apart: the column-wise reads of a wave spread over the banks) and writes 128 bytes of WC rows of
// the result.  Four threads share a column, 32 values each.  WC 64: a scale per column; WC 128: one scale for the block.
template <class T, int WC>
__global__ __launch_bounds__(256) void quantize_transpose_kernel(const T* __restrict__ x, int64_t ld_x, int64_t x_rows, int64_t x_cols, uint8_t* __restrict__ q,
                                                                 int64_t ld_q, uint8_t* __restrict__ scale, int64_t ld_s, unsigned col_tiles) {
    constexpr int LD = WC + 1, PASS = 256 / (WC / 8);          // rows per pass of the workgroup
    extern __shared__ float tile[];
    __shared__ float wave_max[4];
    __shared__ uint8_t bytes[WC];
    const int tid = threadIdx.x;
    // neighbouring tiles of a row of x (which share the lines at their borders) on one die
    const unsigned total = gridDim.x, xcd = blockIdx.x & 7u;
    const unsigned work = xcd * (total >> 3) + min(xcd, total & 7u) + (blockIdx.x >> 3);
    const int64_t r0 = (int64_t)(work / col_tiles) * kBlk, c0 = (int64_t)(work % col_tiles) * WC;
    {
        const int c = tid % (WC / 8) * 8, sub = tid / (WC / 8);
        float v[kBlk / PASS][8];
#pragma unroll
        for (int i = 0; i < kBlk / PASS; ++i) {
            const int64_t row = r0 + i * PASS + sub;
            if (row < x_rows)
                load_run<8>(x + row * ld_x, c0 + c, x_cols, v[i]);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kBlk / PASS; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) tile[(i * PASS + sub) * LD + c + e] = v[i][e];
    }
    __syncthreads();
    const int seg = tid & 3;
    constexpr int COLS = WC / 64;                              // columns per thread
    float amax[COLS];
#pragma unroll
    for (int k = 0; k < COLS; ++k) {
        const int c = (tid >> 2) + k * 64;
        amax[k] = 0.0f;
#pragma unroll
        for (int e = 0; e < 32; ++e) amax[k] = fmaxf(amax[k], finite_magnitude(tile[(seg * 32 + e) * LD + c]));
        amax[k] = fmaxf(amax[k], __shfl_xor(amax[k], 1));
        amax[k] = fmaxf(amax[k], __shfl_xor(amax[k], 2));
    }
    if (WC == 128) {
        float m = fmaxf(amax[0], amax[COLS - 1]);
        for (int o = 4; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        if ((tid & 63) == 0) wave_max[tid >> 6] = m;
        __syncthreads();
        m = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
#pragma unroll
        for (int k = 0; k < COLS; ++k) amax[k] = m;
        if (tid == 0) scale[r0 / kBlk * ld_s + c0 / kBlk] = (uint8_t)scale_byte(m);
    }
#pragma unroll
    for (int k = 0; k < COLS; ++k) {
        const int c = (tid >> 2) + k * 64;
        const unsigned byte = scale_byte(amax[k]);
        const float inv = inverse_scale(byte);
        if (WC == 64 && seg == 0) bytes[c] = (uint8_t)byte;
        if (c0 + c >= x_cols) continue;
        unsigned w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float t[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = no_infinity(tile[(seg * 32 + i * 4 + e) * LD + c] * inv);
            w[i] = pack4_e4m3(t[0], t[1], t[2], t[3]);
        }
        intx4* dst = reinterpret_cast<intx4*>(q + (c0 + c) * ld_q + r0 + seg * 32);
        dst[0] = intx4{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
        dst[1] = intx4{(int)w[4], (int)w[5], (int)w[6], (int)w[7]};
    }
    if (WC == 64) {
        __syncthreads();
        if (tid < 64 && c0 + tid < x_cols) scale[r0 / kBlk * ld_s + c0 + tid] = bytes[tid];
    }
}

struct GemmArgs {
    const uint8_t *a, *as, *b, *bs;
    const float* bias;
    void* c;
    int64_t lda, ldas, ldb, ldbs, ldc;
    int64_t M;
    int N, K;
    bool stream;         // rows of C are whole 128-byte lines: stored past the caches (131072 x 1024 float32 147 -> 113 us; rows that
                         // share lines meet in the L2 instead: 141 us for 16384 x 6719, 188 past it), and partial sums like it
};

// scale byte -> the float whose exponent field it is (what the conversion below reads)
__device__ __forceinline__ float scale_float(int byte) { return byte ? __int_as_float(byte << 23) : __int_as_float(0x00400000); }

// 8 e4m3 values of one row times the block's scale as bfloat16: 4 significant bits, so the conversion is exact (from 2^-130 up to
// 2^128; it rounds to the multiples of 2^-133 that bfloat16 has below, and the products take those)
__device__ __forceinline__ bf16x8 to_bf16(int lo, int hi, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <bool OUT_F32>
__device__ __forceinline__ void store_c(void* c, int64_t at, float v) {
    if (OUT_F32)
        reinterpret_cast<float*>(c)[at] = v;
    else
        reinterpret_cast<__bf16*>(c)[at] = (__bf16)v;
}
// 4 neighbouring columns of a row, of which `left` exist
__device__ __forceinline__ void store_f32x4_edge(float* p, floatx4 v, int left) {
    if (left >= 4) {
        *reinterpret_cast<floatx4_any*>(p) = v;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < left) p[e] = v[e];
}

// ---- few rows of A (M <= 64): bound by reading B once; up to a few MB of it by the latency of a launch and its loads (1 x 6719
// x 256, 1.8 MB: 3.8 us)
//
// A wave owns 16 columns of C (rows of B) for all of M and every waves_k-th block of k; it reads B straight into the
// registers the matrix instruction takes it from (16 whole 128-byte lines per block), so nothing is staged and the loads
// of several blocks are in flight at once.  The waves_k partial sums meet in LDS, added in the order of the waves.
// XT: type of A.  void: quantised operands.  float / uint16_t: values that the wave quantises itself - a lane holds 32
// values of a row, the block's maximum is two lane exchanges away, and the bytes land in the registers the matrix
// instruction reads - which saves linear_fp8 a launch (up to 32 rows, see linear_fp8_fits_rows).
template <class XT, int IM, bool OUT_F32, int BROWS>
__global__ __launch_bounds__(512) void gemm_rows_kernel(GemmArgs g, int waves_k) {
    extern __shared__ float red[];               // [wave][IM][4][64]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wn = wave / waves_k, wk = wave % waves_k, waves_n = (blockDim.x >> 6) / waves_k;
    const int r = lane & 15, kg = lane >> 4;
    const int n0 = (blockIdx.x * waves_n + wn) * 16;
    const int n = n0 + r;
    const int nkb = (g.K + kBlk - 1) / kBlk;
    const bool n_ok = n < g.N;
    const uint8_t* bp = g.b + (int64_t)(n_ok ? n : 0) * g.ldb + kg * 32;
    floatx4 acc[IM] = {};
    for (int kb = wk; kb < nkb; kb += waves_k) {
        intx8 b = *reinterpret_cast<const intx8*>(bp + (int64_t)kb * kBlk);
        const int sb = g.bs[kb * g.ldbs + (n_ok ? n : 0) / BROWS];
        intx8 a[IM];
        int sa[IM];
#pragma unroll
        for (int i = 0; i < IM; ++i) {
            const int m = min(i * 16 + r, (int)g.M - 1);
            if constexpr (__is_same(XT, void)) {
                a[i] = *reinterpret_cast<const intx8*>(g.a + m * g.lda + (int64_t)kb * kBlk + kg * 32);
                sa[i] = g.as[kb * g.ldas + m];
            } else {
                const XT* xp = reinterpret_cast<const XT*>(g.a) + m * g.lda;
                const int k0 = kb * kBlk + kg * 32;
                float v[32], amax = 0.0f;
                load_run<32>(xp, k0, g.K, v);
#pragma unroll
                for (int e = 0; e < 32; ++e) amax = fmaxf(amax, finite_magnitude(v[e]));
                amax = fmaxf(amax, __shfl_xor(amax, 16));
                amax = fmaxf(amax, __shfl_xor(amax, 32));
                sa[i] = (int)scale_byte(amax);
                const float inv = inverse_scale((unsigned)sa[i]);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    a[i][e] = (int)pack4_e4m3(no_infinity(v[4 * e] * inv), no_infinity(v[4 * e + 1] * inv), no_infinity(v[4 * e + 2] * inv), no_infinity(v[4 * e + 3] * inv));
            }
        }
        const float fb = scale_float(sb);
        bf16x8 bv[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) bv[t] = to_bf16(b[2 * t], b[2 * t + 1], fb);
#pragma unroll
        for (int i = 0; i < IM; ++i) {
            const float fa = scale_float(sa[i]);
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bv[t], to_bf16(a[i][2 * t], a[i][2 * t + 1], fa), acc[i], 0, 0, 0);
        }
    }
    // B is the row operand: lane r holds C[i * 16 + r][n0 + 4 kg + e]
    if (waves_k > 1) {
#pragma unroll
        for (int i = 0; i < IM; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[((wave * IM + i) * 4 + e) * 64 + lane] = acc[i][e];
        __syncthreads();
        if (wk != 0) return;
        for (int w = 1; w < waves_k; ++w)
#pragma unroll
            for (int i = 0; i < IM; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][e] += red[(((wave + w) * IM + i) * 4 + e) * 64 + lane];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int no = n0 + kg * 4 + e;
        if (no >= g.N) continue;
        const float bias = g.bias ? g.bias[no] : 0.0f;
#pragma unroll
        for (int i = 0; i < IM; ++i) {
            const int64_t m = i * 16 + r;
            if (m < g.M) store_c<OUT_F32>(g.c, m * g.ldc + no, acc[i][e] + bias);
        }
    }
}

// ---- tiles
//
// A workgroup computes BM x BN of C.  Per block of 128 values of k its rows of A and B (whole 128-byte lines) and A's scale
// bytes go straight from memory to LDS; the next block's copies are in flight while this one is multiplied (two buffers,
// one barrier per block).  A row is 8 pieces of 16 bytes; piece c of row r lies at place c ^ place(r), chosen so that the 16
// lanes of a read phase (lanes 0-3, 12-15 and 20-27 of a half wave, and the other 16) hit 16 different groups of banks; the
// copy writes lane after lane, so the permutation is applied to the address it reads from.  Rows beyond M or N are offsets
// beyond the descriptor: zeros.
// B is the matrix instruction's row operand, A its column operand: a lane then holds 4 neighbouring columns of one row.
//
// Measured: bound by the conversions and matrix instructions beside the operands' loads, 8192^3 into bfloat16 794 to 875 us (1.26
// to 1.38 PFLOP/s; a large bfloat16 library product reaches 1.37), 6719 x 256 x 16384 into float32 73 us (0.78 PFLOP/s with the join of
// 4 pieces).  16384 x 6719 x 256 into float32: 108 us with rows of whole lines (6720 columns apart: 4.1 TB/s, bound by
// writing), 141 us with rows that start anywhere in one, whose ends two tiles write.
struct TileArgs {
    GemmArgs g;
    int tiles_m, tiles_n, splits, kb_split;       // kb_split: blocks of k per split
    float* part;                                  // splits > 1: [split][M][N] partial sums
};

typedef __attribute__((address_space(3))) void* lds_ptr_t;

// (no template parameter may reach the arguments of an LDS-destination load: the host pass would drop the kernel's stub)
__device__ __forceinline__ void copy16(__amdgpu_buffer_rsrc_t rsrc, unsigned char* dst, int voff, int soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)dst, 16, voff, soff, 0, 0);
}
__device__ __forceinline__ void copy4(__amdgpu_buffer_rsrc_t rsrc, unsigned char* dst, int voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)dst, 4, voff, 0, 0, 0);
}

__device__ __forceinline__ int place(int row) { return (row >> 1 & 3) << 1 | (row >> 3 & 1); }

template <int BM, int BN>
constexpr int tile_stage_bytes() { return (BM + BN) * kBlk + 512; }      // operands, then 256 scale bytes of A and of B

// one 16-byte piece of a row of float32 results; STREAM: it leaves the caches first (a result that is not read here)
template <bool STREAM>
__device__ __forceinline__ void store_f32x4(float* p, floatx4 v) {
    if (STREAM)
        __builtin_nontemporal_store(v, reinterpret_cast<floatx4_any*>(p));
    else
        *reinterpret_cast<floatx4_any*>(p) = v;
}
template <bool STREAM>
__device__ __forceinline__ void store_bf16x8(__bf16* p, bf16x8 v) {
    if (STREAM)
        __builtin_nontemporal_store(v, reinterpret_cast<bf16x8_any*>(p));
    else
        *reinterpret_cast<bf16x8_any*>(p) = v;
}

// A workgroup walks its share of the tiles as one sequence of blocks of k: the first block of the next tile is on its way
// while the last of this one is multiplied and the results leave (with a bias, whose loads are issued behind that block's, the
// results wait for it).
template <int BM, int BN, int WGM, int WGN, bool OUT_F32, int BROWS>
__global__ __launch_bounds__(WGM * WGN * 64) void gemm_tile_kernel(TileArgs a) {
    constexpr int WAVES = WGM * WGN, TM = BM / WGM, TN = BN / WGN, IM = TM / 16, IN = TN / 16;
    constexpr int NA = BM / 8, NI = (BM + BN) / 8, PER = NI / WAVES;     // copies of 8 rows: A's, all, per wave
    constexpr int STAGE = tile_stage_bytes<BM, BN>();
    static_assert(NI % WAVES == 0 && BM <= 256 && BN <= 256 && (BROWS == 1 || TN <= 128), "tile");
    constexpr int F32_LANES = TN / 4, F32_STORES = 16 * F32_LANES / 64;  // lanes of a row of results, stores per 16 rows
    constexpr int B16_LANES = TN / 8, B16_STORES = 16 * B16_LANES / 64;
    constexpr int F32_ROW = TN * 4 + 16, B16_ROW = TN * 2 + 16;          // bytes of a staged row
    static_assert(WAVES * 16 * F32_ROW <= STAGE, "staged rows");
    // the fewest stores a full tile's wave makes: a wait that leaves so many operations out waits for everything in front
    constexpr int BEHIND = IM * (OUT_F32 ? F32_STORES : B16_STORES);
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const GemmArgs& g = a.g;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WGN, wn = wave % WGN;
    const int r = lane & 15, kg = lane >> 4;
    const int nkb = (g.K + kBlk - 1) / kBlk;
    const bool partial = a.splits > 1;

    // Workgroups go to the 8 dies in turn: every die gets a contiguous range of the tiles, its workgroups take them in
    // turn, in bands of 8 tile rows, so that what a die computes at one time shares rows of A and B in its L2.
    const unsigned total = (unsigned)a.tiles_m * a.tiles_n * a.splits, xcd = blockIdx.x & 7u;
    const unsigned lo = xcd * (total >> 3) + min(xcd, total & 7u), hi = lo + (total >> 3) + (xcd < (total & 7u) ? 1u : 0u);
    const unsigned stride = (gridDim.x >> 3) + (xcd < (gridDim.x & 7u) ? 1u : 0u);       // workgroups of this die
    unsigned job = lo + (blockIdx.x >> 3);
    if (job >= hi) return;
    struct Job {
        int64_t m0;
        int n0, kb0, kb1, split;
    };
    auto job_of = [&](unsigned work) {
        Job j;
        const unsigned per_split = (unsigned)a.tiles_m * a.tiles_n;
        j.split = (int)(work / per_split);
        work %= per_split;
        const unsigned band = work / (8u * a.tiles_n), rows_in_band = min(8u, a.tiles_m - band * 8);
        const unsigned in_band = work - band * 8u * a.tiles_n;
        j.m0 = (int64_t)(band * 8 + in_band % rows_in_band) * BM;
        j.n0 = (int)(in_band / rows_in_band) * BN;
        j.kb0 = j.split * a.kb_split;
        j.kb1 = min(nkb, j.kb0 + a.kb_split);
        return j;
    };

    // ---- the tile whose operands are being fetched
    Job in = job_of(job);
    __amdgpu_buffer_rsrc_t ra, rb;
    int src[PER];
    int64_t sb_col = 0;
    auto open = [&] {
        const int rows_a = (int)min((int64_t)BM, g.M - in.m0), rows_b = min(BN, g.N - in.n0), k_bytes = (in.kb1 - in.kb0) * kBlk;
        ra = __builtin_amdgcn_make_buffer_rsrc((void*)(g.a + in.m0 * g.lda + (int64_t)in.kb0 * kBlk), 0, (unsigned)((rows_a - 1) * (int)g.lda + k_bytes), 0x00020000);
        rb = __builtin_amdgcn_make_buffer_rsrc((void*)(g.b + in.n0 * g.ldb + (int64_t)in.kb0 * kBlk), 0, (unsigned)((rows_b - 1) * (int)g.ldb + k_bytes), 0x00020000);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = wave * PER + i;
            const int row = (c < NA ? c : c - NA) * 8 + (lane >> 3);
            const int piece = (lane & 7) ^ place(row);
            const bool ok = row < (c < NA ? rows_a : rows_b);
            src[i] = ok ? row * (int)(c < NA ? g.lda : g.ldb) + piece * 16 : (int)0x80000000;
        }
        // the wave's columns lie within one block of 128: its scale is a scalar load
        sb_col = min(in.n0 + wn * TN, g.N - 1) / kBlk;
    };
    auto issue = [&](int kb, int half) {
        unsigned char* base = lds + half * STAGE;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = wave * PER + i;
            copy16(c < NA ? ra : rb, base + c * 1024, src[i], (kb - in.kb0) * kBlk);
        }
        if (wave == 0) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(g.as + (int64_t)kb * g.ldas + in.m0), 0, (unsigned)scale_window(BM, g.M, in.m0), 0x00020000);
            copy4(rs, base + (BM + BN) * kBlk, lane * 4);
        }
        if (BROWS == 1 && wave == WAVES - 1) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(g.bs + (int64_t)kb * g.ldbs + in.n0), 0, (unsigned)scale_window(BN, g.N, in.n0), 0x00020000);
            copy4(rs, base + (BM + BN) * kBlk + 256, lane * 4);
        }
    };
    open();
    int kb_in = in.kb0, half = 0;
    issue(kb_in, 0);
    int sb_next = BROWS == 1 ? 0 : g.bs[(int64_t)kb_in * g.ldbs + sb_col];

    // ---- the tile that is being multiplied
    Job out = in;
    bool more = true;                                   // blocks left to fetch
    bool behind = false;                                // BEHIND stores or more have been issued since the last copies
    const int a_row = wm * TM + r, b_row = wn * TN + r;
    for (;;) {
    floatx4 acc[IM][IN];
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int kb = out.kb0; kb < out.kb1; ++kb, half ^= 1) {
        // my copies have landed and my reads of the other buffer are done; behind the barrier everybody's
        if (behind)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(BEHIND) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        behind = false;
        const int sb = sb_next;
        if (++kb_in == in.kb1) {
            job += stride;
            more = job < hi;
            if (more) {
                in = job_of(job);
                open();
                kb_in = in.kb0;
            }
        }
        if (more) {
            issue(kb_in, half ^ 1);
            if (BROWS != 1) sb_next = g.bs[(int64_t)kb_in * g.ldbs + sb_col];
        }
        const unsigned char* base = lds + half * STAGE;
        const unsigned char* pa = base + a_row * kBlk;
        const unsigned char* pb = base + (BM + b_row) * kBlk;
        const unsigned char* psa = base + (BM + BN) * kBlk + a_row;
        const unsigned char* psb = base + (BM + BN) * kBlk + 256 + b_row;
        const int sw = place(r);                        // rows 16 apart have the same permutation
#pragma unroll
        for (int h = 0; h < 2; ++h) {                   // 16 of the lane's 32 bytes: two instructions of 32 values of k
            const int at = ((2 * kg + h) ^ sw) * 16;
            bf16x8 bv[IN][2];
#pragma unroll
            for (int j = 0; j < IN; ++j) {
                const intx4 q = *reinterpret_cast<const intx4*>(pb + j * 16 * kBlk + at);
                const float f = scale_float(BROWS == 1 ? (int)psb[j * 16] : sb);
                bv[j][0] = to_bf16(q[0], q[1], f);
                bv[j][1] = to_bf16(q[2], q[3], f);
            }
#pragma unroll
            for (int i = 0; i < IM; ++i) {
                const intx4 q = *reinterpret_cast<const intx4*>(pa + i * 16 * kBlk + at);
                const float f = scale_float((int)psa[i * 16]);
                const bf16x8 a0 = to_bf16(q[0], q[1], f), a1 = to_bf16(q[2], q[3], f);
#pragma unroll
                for (int j = 0; j < IN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bv[j][0], a0, acc[i][j], 0, 0, 0);
#pragma unroll
                for (int j = 0; j < IN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bv[j][1], a1, acc[i][j], 0, 0, 0);
            }
        }
    }
    {
        const int used = half ^ 1;                      // the buffer of the last block
        // Lane (r, kg) holds C[m0 + wm TM + 16 i + r][n0 + wn TN + 16 j + 4 kg .. + 3]: 16 bytes of 16 rows per store.  Every
        // wave turns its 16-row slices through an area of its own in the buffer just used into runs of whole rows of its
        // TN columns, which fill the lines they touch (rows of odd length start anywhere in one).
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();                   // every wave is done with that buffer's operands
        asm volatile("" ::: "memory");
        const bool full = out.m0 + BM <= g.M && out.n0 + BN <= g.N;
        if (partial || OUT_F32) {
            unsigned char* mine = lds + used * STAGE + wave * (16 * F32_ROW);
            const int64_t ldo = partial ? g.N : g.ldc;
            const int c4 = lane % F32_LANES * 4, n = out.n0 + wn * TN + c4;
            const int64_t m_first = out.m0 + wm * TM + lane / F32_LANES;
            float* dst = (partial ? a.part + (int64_t)out.split * g.M * g.N : reinterpret_cast<float*>(g.c)) + m_first * ldo + n;
            floatx4 bias = {0.0f, 0.0f, 0.0f, 0.0f};
            if (g.bias && !partial)
#pragma unroll
                for (int e = 0; e < 4; ++e) bias[e] = n + e < g.N ? g.bias[n + e] : 0.0f;
#pragma unroll
            for (int i = 0; i < IM; ++i) {
#pragma unroll
                for (int j = 0; j < IN; ++j) *reinterpret_cast<floatx4*>(mine + r * F32_ROW + (j * 16 + kg * 4) * 4) = acc[i][j];
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int t = 0; t < F32_STORES; ++t) {
                    constexpr int STEP = 64 / F32_LANES;
                    const floatx4 v = *reinterpret_cast<const floatx4*>(mine + (t * STEP + lane / F32_LANES) * F32_ROW + c4 * 4) + bias;
                    float* at = dst + (i * 16 + t * STEP) * ldo;
                    if (full && g.stream)
                        store_f32x4<true>(at, v);
                    else if (full)
                        store_f32x4<false>(at, v);
                    else if (m_first + i * 16 + t * STEP < g.M)
                        store_f32x4_edge(at, v, g.N - n);
                }
                __builtin_amdgcn_wave_barrier();
            }
        } else {
            unsigned char* mine = lds + used * STAGE + wave * (16 * B16_ROW);
            const int c8 = lane % B16_LANES * 8, n8 = out.n0 + wn * TN + c8;
            const int64_t m_first = out.m0 + wm * TM + lane / B16_LANES;
            __bf16* dst = reinterpret_cast<__bf16*>(g.c) + m_first * g.ldc + n8;
#pragma unroll
            for (int i = 0; i < IM; ++i) {
#pragma unroll
                for (int j = 0; j < IN; ++j) {
                    const int n = out.n0 + wn * TN + j * 16 + kg * 4;
                    floatx4 v = acc[i][j];
                    if (g.bias)
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] += n + e < g.N ? g.bias[n + e] : 0.0f;
                    *reinterpret_cast<bf16x4*>(mine + r * B16_ROW + (j * 16 + kg * 4) * 2) = bf16x4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
                }
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int t = 0; t < B16_STORES; ++t) {
                    constexpr int STEP = 64 / B16_LANES;
                    const bf16x8 v = *reinterpret_cast<const bf16x8*>(mine + (t * STEP + lane / B16_LANES) * B16_ROW + c8 * 2);
                    __bf16* at = dst + (i * 16 + t * STEP) * g.ldc;
                    if (full && g.stream) {
                        store_bf16x8<true>(at, v);
                    } else if (full) {
                        store_bf16x8<false>(at, v);
                    } else if (m_first + i * 16 + t * STEP < g.M) {
                        if (n8 + 8 <= g.N) {
                            *reinterpret_cast<bf16x8_any*>(at) = v;
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (n8 + e < g.N) at[e] = v[e];
                        }
                    }
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
        if (!more) return;
        behind = full;
        out = in;
    }
    }
}

// The partial sums of the splits, in their order, and the bias.  BATCH loads are in flight: 4 for few splits (more cost
// occupancy: 6719 x 256 with 4 splits 72 us with the product, 76 with 16 in flight), 16 for many (65 x 64 with 64: 18 against
// 31).
template <bool OUT_F32, int BATCH>
__global__ __launch_bounds__(256) void gemm_join_kernel(const float* __restrict__ part, int splits, int64_t M, int N, const float* __restrict__ bias, void* c, int64_t ldc) {
    const int64_t count = M * N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        float v = part[i];
        for (int z = 1; z < splits; z += BATCH) {
            float t[BATCH];
#pragma unroll
            for (int u = 0; u < BATCH; ++u) t[u] = part[min(z + u, splits - 1) * count + i];
#pragma unroll
            for (int u = 0; u < BATCH; ++u)
                if (z + u < splits) v += t[u];
        }
        const int64_t m = i / N;
        const int n = (int)(i - m * N);
        store_c<OUT_F32>(c, m * ldc + n, v + (bias ? bias[n] : 0.0f));
    }
}

template <int BM, int BN, int WGM, int WGN, bool OUT_F32, int BROWS>
int launch_tile(const TileArgs& a, hipStream_t s) {
    constexpr int bytes = 2 * tile_stage_bytes<BM, BN>();
    OCR_REQUIRE(a.tiles_m == (a.g.M + BM - 1) / BM && a.tiles_n == (a.g.N + BN - 1) / BN && a.splits >= 1 &&
                    (int64_t)(a.splits - 1) * a.kb_split < (a.g.K + kBlk - 1) / kBlk,
                "gemm_fp8: %d x %d tiles and %d splits do not fit the kernel", a.tiles_m, a.tiles_n, a.splits);
    auto kernel = &gemm_tile_kernel<BM, BN, WGM, WGN, OUT_F32, BROWS>;
    static bool opted[64] = {};
    int dev = 0;
    OCR_HIP_CHECK(hipGetDevice(&dev));
    {
        std::lock_guard<std::mutex> lock(g_lds_mutex);
        if (!opted[dev & 63]) {
            OCR_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
            opted[dev & 63] = true;
        }
    }
    hipLaunchKernelGGL((gemm_tile_kernel<BM, BN, WGM, WGN, OUT_F32, BROWS>), dim3((unsigned)std::min<int64_t>((int64_t)a.tiles_m * a.tiles_n * a.splits, BM * BN > 128 * 128 ? 256 : 512)), dim3(WGM * WGN * 64), bytes, s, a);
    OCR_HIP_CHECK(hipGetLastError());
    return OCRHIP_OK;
}

struct TilePlan {
    int bm, bn, splits, kb_split;
    int64_t tiles_m, tiles_n;
};

// Which tiles a product of M > kMaxRows rows takes, and into how many pieces of k it is split.
//
// Tiles of 256 x 256 (bfloat16 results; one workgroup per compute unit) read their operands half as often.  They win where
// they fill their rounds of the 256 compute units to nine tenths (8192^3 875 us against 976 of 128 x 128, 4096^3 108 against
// 115, 131072 x 1024 x 256 85 against 92) and lose where the last round leaves compute units idle (5000 x 5000 x 640, 400 tiles,
// 44 against 40; 79872 x 256 x 512, 312 tiles, 36 against 25; 4096 x 3200 x 512, 208 tiles, 22 against 20).  float32 results
// take 128 x 128 throughout.
//
// Pieces of k (both result types run the same loop): a workgroup takes 1.05 us per block of k as long as it has its compute
// unit to itself and 1.6 us when two share one; joining the pieces costs a launch, 2.5 us, and 0.27 us per MB of partial sums
// (written and read).  What comes out least is taken, up to two workgroups per compute unit, for the 513th would make a second round of them all.  Measured
// against one piece: 300 x 97 x 2048 10 us / 22, 256 x 256 x 131072 33 / 1087, 6719 x 256 x 16384 73 / 142; where one piece
// stays, against two: 1900 x 1900 x 2048 26 / 32, 1000 x 1000 x 1024 14 / 16.
TilePlan plan_tiles(int64_t M, int64_t N, int64_t K, bool out_f32) {
    TilePlan p;
    const int64_t nkb = (K + kBlk - 1) / kBlk;
    const int64_t big = ((M + 255) / 256) * ((N + 255) / 256);
    const bool large = !out_f32 && 10 * big >= 9 * 256 * ((big + 255) / 256);
    p.bm = large ? 256 : 128;
    p.bn = large ? 256 : 128;
    p.tiles_m = (M + p.bm - 1) / p.bm;
    p.tiles_n = (N + p.bn - 1) / p.bn;
    const int64_t tiles = p.tiles_m * p.tiles_n;
    p.splits = 1;
    p.kb_split = (int)nkb;
    double least = 1.05 * (double)nkb;
    const int64_t most = large ? 1 : std::min<int64_t>(nkb, 512 / std::max<int64_t>(tiles, 1));
    for (int64_t s = 2; s <= most; s += s < 4 ? 1 : s / 2) {
        const int64_t per = (nkb + s - 1) / s, pieces = (nkb + per - 1) / per;
        const double us = (pieces * tiles <= 256 ? 1.05 : 1.6) * (double)per + 2.5 + 0.27e-6 * 8.0 * (double)(pieces * M * N);
        if (us < least) {
            least = us;
            p.splits = (int)pieces;
            p.kb_split = (int)per;
        }
    }
    return p;
}

template <class XT, bool OUT_F32, int BROWS>
int launch_rows(const GemmArgs& g, hipStream_t s) {
    const int nkb = (g.K + kBlk - 1) / kBlk;
    int waves_k = 1;
    while (waves_k < 8 && waves_k * 2 <= nkb) waves_k *= 2;
    const int waves_n = std::max(1, 4 / waves_k);
    const int waves = waves_k * waves_n, im = (int)((g.M + 15) / 16);
    const dim3 grid((unsigned)((g.N + 16 * waves_n - 1) / (16 * waves_n))), block(waves * 64);
    const size_t lds = waves_k > 1 ? (size_t)waves * im * 4 * 64 * sizeof(float) : 0;
    switch (im) {
        case 1: hipLaunchKernelGGL((gemm_rows_kernel<XT, 1, OUT_F32, BROWS>), grid, block, lds, s, g, waves_k); break;
        case 2: hipLaunchKernelGGL((gemm_rows_kernel<XT, 2, OUT_F32, BROWS>), grid, block, lds, s, g, waves_k); break;
        case 3:
            if constexpr (__is_same(XT, void)) hipLaunchKernelGGL((gemm_rows_kernel<XT, 3, OUT_F32, BROWS>), grid, block, lds, s, g, waves_k);
            break;
        default:
            if constexpr (__is_same(XT, void)) hipLaunchKernelGGL((gemm_rows_kernel<XT, 4, OUT_F32, BROWS>), grid, block, lds, s, g, waves_k);
            break;
    }
    OCR_HIP_CHECK(hipGetLastError());
    return OCRHIP_OK;
}

template <class XT>
int launch_rows_any(const GemmArgs& g, bool f32, int b_block_rows, hipStream_t s) {
    if (b_block_rows == 1) return f32 ? launch_rows<XT, true, 1>(g, s) : launch_rows<XT, false, 1>(g, s);
    return f32 ? launch_rows<XT, true, kBlk>(g, s) : launch_rows<XT, false, kBlk>(g, s);
}

// gemm_rows_kernel up to 64 rows of A (64 x 6719 x 256: 6.4 us against 7.3 of tiles, 64 x 1024 x 2048 9.7 against 11.5)
constexpr int kMaxRows = 64;

template <class T>
int launch_quantize(const T* x, int64_t rows, int64_t cols, int64_t ld_x, int block_rows, bool transpose, uint8_t* q, int64_t ld_q, uint8_t* scale,
                    int64_t ld_s, hipStream_t s) {
    const int64_t nkb = (cols + kBlk - 1) / kBlk, nrb = (rows + kBlk - 1) / kBlk;
    int64_t grid;
    if (transpose) {
        const int wc = block_rows == 1 ? 64 : 128;
        const int64_t col_tiles = (cols + wc - 1) / wc;
        grid = nrb * col_tiles;
        OCR_REQUIRE(grid * 256 < (1ll << 32), "quantize_fp8: too many blocks");
        const size_t lds = (size_t)kBlk * (wc + 1) * sizeof(float);
        if (wc == 64) {
            hipLaunchKernelGGL((quantize_transpose_kernel<T, 64>), dim3((unsigned)grid), dim3(256), lds, s, x, ld_x, rows, cols, q, ld_q, scale, ld_s, (unsigned)col_tiles);
        } else {
            static bool opted[64] = {};
            int dev = 0;
            OCR_HIP_CHECK(hipGetDevice(&dev));
            std::lock_guard<std::mutex> lock(g_lds_mutex);
            if (!opted[dev & 63]) {
                OCR_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(&quantize_transpose_kernel<T, 128>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
                opted[dev & 63] = true;
            }
            hipLaunchKernelGGL((quantize_transpose_kernel<T, 128>), dim3((unsigned)grid), dim3(256), lds, s, x, ld_x, rows, cols, q, ld_q, scale, ld_s, (unsigned)col_tiles);
        }
    } else if (block_rows == 1) {
        const int64_t chunks = (nkb + kBlocksWg - 1) / kBlocksWg;
        grid = (rows + kRowsWg - 1) / kRowsWg * chunks;
        OCR_REQUIRE(grid * 256 < (1ll << 32), "quantize_fp8: too many blocks");
        hipLaunchKernelGGL(quantize_rows_kernel<T>, dim3((unsigned)grid), dim3(256), 0, s, x, ld_x, rows, cols, q, ld_q, scale, ld_s, (unsigned)chunks);
    } else {
        grid = nrb * nkb;
        OCR_REQUIRE(grid * 256 < (1ll << 32), "quantize_fp8: too many blocks");
        hipLaunchKernelGGL(quantize_block_kernel<T>, dim3((unsigned)grid), dim3(256), 0, s, x, ld_x, rows, cols, q, ld_q, scale, ld_s, (unsigned)nkb);
    }
    OCR_HIP_CHECK(hipGetLastError());
    return OCRHIP_OK;
}

}  // namespace

int launch_quantize_fp8(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ld_x, int block_rows, bool transpose,
                        uint8_t* q, int64_t ld_q, uint8_t* scale, int64_t ld_scale, hipStream_t s) {
    const int64_t R = transpose ? cols : rows, C = transpose ? rows : cols;
    if (R == 0 || C == 0) return OCRHIP_OK;
    const int64_t rb = (R + block_rows - 1) / block_rows, cb = (C + kBlk - 1) / kBlk;
    const double n = (double)rows * cols;
    ProfScope prof(transpose ? "quantize_fp8<t>" : "quantize_fp8", 2.0 * n, n * ((x_dtype == OCRHIP_F32 ? 4.0 : 2.0) + 1.0) + (double)rb * cb, s);
    return x_dtype == OCRHIP_F32 ? launch_quantize((const float*)x, rows, cols, ld_x, block_rows, transpose, q, ld_q, scale, ld_scale, s)
                                 : launch_quantize((const uint16_t*)x, rows, cols, ld_x, block_rows, transpose, q, ld_q, scale, ld_scale, s);
}

size_t gemm_fp8_workspace(int64_t M, int64_t N, int64_t K) {
    if (M <= kMaxRows) return 0;
    const int a = plan_tiles(M, N, K, true).splits, b = plan_tiles(M, N, K, false).splits, splits = std::max(a, b);
    return splits > 1 ? (size_t)splits * M * N * sizeof(float) : 0;
}

int launch_gemm_fp8(const Fp8Operand& a, const Fp8Operand& b, int b_block_rows, int64_t M, int64_t N, int64_t K, const float* bias,
                    void* c, int c_dtype, int64_t ld_c, void* ws, hipStream_t s) {
    if (M == 0 || N == 0) return OCRHIP_OK;
    const bool f32 = c_dtype == OCRHIP_F32;
    const int64_t row_bytes = ld_c * (f32 ? 4 : 2);
    GemmArgs g{a.q, a.scale, b.q, b.scale, bias, c, a.ld, a.ld_scale, b.ld, b.ld_scale, ld_c, M, (int)N, (int)K, row_bytes % 128 == 0 && reinterpret_cast<uintptr_t>(c) % 128 == 0};
    const double flops = 2.0 * (double)M * N * K, bytes = (double)(M + N) * K + (f32 ? 4.0 : 2.0) * (double)M * N;
    if (M <= kMaxRows) {
        ProfScope prof(f32 ? "gemm_fp8<rows,f32>" : "gemm_fp8<rows,bf16>", flops, bytes, s);
        return launch_rows_any<void>(g, f32, b_block_rows, s);
    }
    const TilePlan p = plan_tiles(M, N, K, f32);
    OCR_REQUIRE(p.tiles_m * p.tiles_n * p.splits < (1ll << 31), "gemm_fp8: too many tiles");
    TileArgs t{g, (int)p.tiles_m, (int)p.tiles_n, p.splits, p.kb_split, reinterpret_cast<float*>(ws)};
    {
        ProfScope prof(p.bm == 256 ? "gemm_fp8<256,bf16>" : f32 ? "gemm_fp8<128,f32>" : "gemm_fp8<128,bf16>", flops, bytes, s);
        if (f32)
            OCR_TRY(b_block_rows == 1 ? (launch_tile<128, 128, 2, 2, true, 1>(t, s)) : (launch_tile<128, 128, 2, 2, true, kBlk>(t, s)));
        else if (p.bm == 256)
            OCR_TRY(b_block_rows == 1 ? (launch_tile<256, 256, 2, 4, false, 1>(t, s)) : (launch_tile<256, 256, 2, 4, false, kBlk>(t, s)));
        else
            OCR_TRY(b_block_rows == 1 ? (launch_tile<128, 128, 2, 2, false, 1>(t, s)) : (launch_tile<128, 128, 2, 2, false, kBlk>(t, s)));
    }
    if (p.splits > 1) {
        ProfScope prof("gemm_fp8<join>", (double)p.splits * M * N, ((f32 ? 4.0 : 2.0) + 4.0 * p.splits) * (double)M * N, s);
        const dim3 grid((unsigned)std::min<int64_t>((M * N + 255) / 256, 4096));
        auto join = f32 ? (p.splits > 16 ? &gemm_join_kernel<true, 16> : &gemm_join_kernel<true, 4>) : (p.splits > 16 ? &gemm_join_kernel<false, 16> : &gemm_join_kernel<false, 4>);
        hipLaunchKernelGGL(join, grid, dim3(256), 0, s, t.part, p.splits, M, (int)N, bias, c, ld_c);
        OCR_HIP_CHECK(hipGetLastError());
    }
    return OCRHIP_OK;
}

// Whether the kernel for few rows quantises them itself.  Up to 16 rows that saves the launch (1 x 6719 x 256: 3.8 us against
// 5.5, 16 x 1024 x 2048 7.8 against 8.2); with 32 every wave quantises twice as much of each block, which costs more than the
// launch when k is long (32 x 6719 x 256: 6.6 against 7.1; 32 x 1024 x 2048: 12.3 against 9.8).
bool linear_fp8_fits_rows(int64_t M, int64_t K) { return M <= 16 || (M <= 32 && K <= 512); }

int launch_linear_fp8_rows(const void* x, int x_dtype, int64_t ld_x, const Fp8Operand& b, int b_block_rows, int64_t M, int64_t N, int64_t K, const float* bias,
                           void* c, int c_dtype, int64_t ld_c, hipStream_t s) {
    if (M == 0 || N == 0) return OCRHIP_OK;
    const bool f32 = c_dtype == OCRHIP_F32, xf32 = x_dtype == OCRHIP_F32;
    GemmArgs g{reinterpret_cast<const uint8_t*>(x), nullptr, b.q, b.scale, bias, c, ld_x, 0, b.ld, b.ld_scale, ld_c, M, (int)N, (int)K, false};
    ProfScope prof("linear_fp8<rows>", 2.0 * (double)M * N * K, (xf32 ? 4.0 : 2.0) * (double)M * K + (double)N * K + (f32 ? 4.0 : 2.0) * (double)M * N, s);
    return xf32 ? launch_rows_any<float>(g, f32, b_block_rows, s) : launch_rows_any<uint16_t>(g, f32, b_block_rows, s);
}

}  // namespace ocrhip
