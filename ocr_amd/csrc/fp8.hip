// 8-bit floating point products with a scale for each block of 128 (no counterpart in the reference, which computes in
// float32).
//
//   quantise:  the values of a block (1 x 128, or 128 x 128 of a weight matrix) are divided by a power of two 2^e, the
//              least with amax <= 448 * 2^e (448 is the largest e4m3 value), and rounded to e4m3 (nearest, ties to even):
//              the division is exact, so the only rounding is that to four significant bits.
//   product:   C[m,n] = sum over blocks j of 2^(ea[m,j] + eb[n,j]) * sum over k in j of A[m,k] * B[n,k]  (+ bias[n])
//
// The scales are powers of two because the matrix instruction takes those itself (one exponent byte per row and 32 values
// of k): the products of all blocks then add up in ONE float32 accumulator, without a multiply-add of every accumulator by
// a float scale after each block.  A float scale would use the range of e4m3 better by less than a factor of 2, which a
// floating type does not need: the relative rounding error is 2^-4 at any magnitude.
//
// Two forms of the product, chosen by the type of the result:
//   bfloat16 result: v_mfma_scale_f32_16x16x128_f8f6f4 on the bytes.  The 8-bit matrix instructions add the products of a
//     group of neighbouring values of k (at most 16) aligned to the largest of them and keep 13 bits below it (measured: a
//     product 2^-14 of its neighbour's is lost, one 16 places further is not; group sums and the accumulator are float32).
//     That is 1e-4 of the result at most for ordinary data, a fortieth of the rounding to bfloat16 that follows.
//   float32 result: the bytes times their scale are converted to bfloat16 on the way from LDS (exact: 4 significant bits)
//     and multiplied by v_mfma_f32_16x16x32_bf16, which keeps float32 throughout, at half the rate.
#include <cmath>

#include "common.h"

namespace ocrhip {

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

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

// 2^-(byte - 127) as a product of two floats: 2^127 is one, but the factor of a byte 0 block's subnormals is 2^127 and the
// one of byte 247 is 2^-120, so one float holds every factor that occurs.
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

template <class T>
__global__ __launch_bounds__(256) void quantize_simple_kernel(const T* __restrict__ x, int64_t ld_x, int64_t rows, int64_t cols, int block_rows,
                                                              int transpose, uint8_t* __restrict__ q, int64_t ld_q,
                                                              uint8_t* __restrict__ scale, int64_t ld_s) {
    __shared__ float part[4];
    const int64_t rb = blockIdx.x, cb = blockIdx.y;
    const int tid = threadIdx.x;
    const int64_t r0 = rb * block_rows, c0 = cb * kBlk;
    const int nr = (int)min((int64_t)block_rows, rows - r0);
    auto value = [&](int r, int c) -> float {
        if (c0 + c >= cols) return 0.0f;
        return load_f32(transpose ? x + (c0 + c) * ld_x + r0 + r : x + (r0 + r) * ld_x + c0 + c);
    };
    float amax = 0.0f;
    for (int i = tid; i < nr * kBlk; i += 256) amax = fmaxf(amax, finite_magnitude(value(i / kBlk, i % kBlk)));
    for (int o = 32; o; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    if ((tid & 63) == 0) part[tid >> 6] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    const unsigned byte = scale_byte(amax);
    const float inv = inverse_scale(byte);
    if (tid == 0) scale[cb * ld_s + rb] = (uint8_t)byte;
    for (int i = tid; i < nr * (kBlk / 4); i += 256) {
        const int r = i / (kBlk / 4), c = i % (kBlk / 4) * 4;
        float v[4];
        for (int e = 0; e < 4; ++e) v[e] = no_infinity(value(r, c + e) * inv);
        *reinterpret_cast<unsigned*>(q + (r0 + r) * ld_q + c0 + c) = pack4_e4m3(v[0], v[1], v[2], v[3]);
    }
}

struct GemmArgs {
    const uint8_t *a, *as, *b, *bs;
    const float* bias;
    void* c;
    int64_t lda, ldas, ldb, ldbs, ldc;
    int64_t M;
    int N, K;
};

// scale byte -> the float whose exponent field it is (what the conversion below reads)
__device__ __forceinline__ float scale_float(int byte) { return byte ? __int_as_float(byte << 23) : __int_as_float(0x00400000); }

// 8 e4m3 values of one row times the block's scale as bfloat16: 4 significant bits, so the conversion is exact
__device__ __forceinline__ bf16x8 to_bf16(int lo, int hi, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// wave: 16 rows x 64 columns, operands straight from memory in the layout the instruction reads (lane: row l % 16, the 32
// bytes of k group l / 16; the group's order inside the 128 values does not matter, as A and B have the same)
template <int BROWS, bool OUT_F32>
__global__ __launch_bounds__(256) void gemm_simple_kernel(GemmArgs g) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t m0 = (int64_t)blockIdx.x * 64 + wave * 16;
    const int n0 = blockIdx.y * 64;
    const int r = lane & 15, kg = lane >> 4;
    const int64_t m = m0 + r;
    floatx4 acc[4] = {};
    const int nkb = (g.K + kBlk - 1) / kBlk;
    for (int kb = 0; kb < nkb; ++kb) {
        intx8 a = {};
        int sa = kBias;
        if (m < g.M) {
            a = *reinterpret_cast<const intx8*>(g.a + m * g.lda + (int64_t)kb * kBlk + kg * 32);
            sa = g.as[kb * g.ldas + m];
        }
        const float fa = scale_float(sa);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int n = n0 + t * 16 + r;
            intx8 b = {};
            int sb = kBias;
            if (n < g.N) {
                b = *reinterpret_cast<const intx8*>(g.b + (int64_t)n * g.ldb + (int64_t)kb * kBlk + kg * 32);
                sb = g.bs[kb * g.ldbs + n / BROWS];
            }
            if constexpr (OUT_F32) {
                const float fb = scale_float(sb);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(a[2 * i], a[2 * i + 1], fa), to_bf16(b[2 * i], b[2 * i + 1], fb), acc[t], 0, 0, 0);
            } else {
                acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc[t], 0, 0, 0, sa, 0, sb);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int n = n0 + t * 16 + r;
        if (n >= g.N) continue;
        const float bias = g.bias ? g.bias[n] : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t mo = m0 + kg * 4 + e;
            if (mo >= g.M) continue;
            const float v = acc[t][e] + bias;
            if (OUT_F32)
                reinterpret_cast<float*>(g.c)[mo * g.ldc + n] = v;
            else
                reinterpret_cast<__bf16*>(g.c)[mo * g.ldc + n] = (__bf16)v;
        }
    }
}

}  // namespace

int launch_quantize_fp8(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ld_x, int block_rows, bool transpose,
                        uint8_t* q, int64_t ld_q, uint8_t* scale, int64_t ld_scale, hipStream_t s) {
    const int64_t R = transpose ? cols : rows, C = transpose ? rows : cols;
    if (R == 0 || C == 0) return OCRHIP_OK;
    const int64_t rb = (R + block_rows - 1) / block_rows, cb = (C + kBlk - 1) / kBlk;
    const double n = (double)rows * cols;
    ProfScope prof(transpose ? "quantize_fp8<t>" : "quantize_fp8", 2.0 * n, n * ((x_dtype == OCRHIP_F32 ? 4.0 : 2.0) + 1.0) + (double)rb * cb, s);
    const dim3 grid((unsigned)rb, (unsigned)cb);
    if (x_dtype == OCRHIP_F32)
        hipLaunchKernelGGL(quantize_simple_kernel<float>, grid, dim3(256), 0, s, (const float*)x, ld_x, R, C, block_rows, transpose ? 1 : 0, q, ld_q, scale, ld_scale);
    else
        hipLaunchKernelGGL(quantize_simple_kernel<uint16_t>, grid, dim3(256), 0, s, (const uint16_t*)x, ld_x, R, C, block_rows, transpose ? 1 : 0, q, ld_q, scale, ld_scale);
    OCR_HIP_CHECK(hipGetLastError());
    return OCRHIP_OK;
}

size_t gemm_fp8_workspace(int64_t M, int64_t N, int64_t K) {
    (void)M; (void)N; (void)K;
    return 0;
}

int launch_gemm_fp8(const Fp8Operand& a, const Fp8Operand& b, int b_block_rows, int64_t M, int64_t N, int64_t K, const float* bias,
                    void* c, int c_dtype, int64_t ld_c, void* ws, hipStream_t s) {
    (void)ws;
    if (M == 0 || N == 0) return OCRHIP_OK;
    GemmArgs g{a.q, a.scale, b.q, b.scale, bias, c, a.ld, a.ld_scale, b.ld, b.ld_scale, ld_c, M, (int)N, (int)K};
    const bool f32 = c_dtype == OCRHIP_F32;
    ProfScope prof("gemm_fp8", 2.0 * (double)M * N * K, (double)(M + N) * K + (f32 ? 4.0 : 2.0) * (double)M * N, s);
    const dim3 grid((unsigned)((M + 63) / 64), (unsigned)((N + 63) / 64));
    if (b_block_rows == 1) {
        if (f32) hipLaunchKernelGGL((gemm_simple_kernel<1, true>), grid, dim3(256), 0, s, g);
        else hipLaunchKernelGGL((gemm_simple_kernel<1, false>), grid, dim3(256), 0, s, g);
    } else {
        if (f32) hipLaunchKernelGGL((gemm_simple_kernel<kBlk, true>), grid, dim3(256), 0, s, g);
        else hipLaunchKernelGGL((gemm_simple_kernel<kBlk, false>), grid, dim3(256), 0, s, g);
    }
    OCR_HIP_CHECK(hipGetLastError());
    return OCRHIP_OK;
}

}  // namespace ocrhip
