// Distillation from a teacher's top logits (no counterpart in the reference, which holds no training code for this path):
// the K largest logits of a row with its log normaliser (the teacher's side), and the loss of a student's logits against
// them with its gradient.
//
//   entries k of a row: class i_k, logit z_k; temperature tau; student logits s
//   p_k = softmax of z / tau over the entries, or, with the teacher's lse = log sum_v exp(z_v / tau),
//   p_k = exp(z_k / tau - lse) and one more class p_rest = 1 - sum p_k for everything outside the entries
//   q   = softmax(s / tau);  q_rest = sum of q outside the entries
//   loss = w tau^2 (sum_k p_k log(p_k / q_(i_k)) [+ p_rest log(p_rest / q_rest)])
//   d loss / d s_v = w tau (P q_v - p_v) for the entries, w tau q_v (P [- p_rest / q_rest]) outside them, P = sum_k p_k
//   [+ p_rest], which is 1 but where the entries' mass exceeds it or they name every class
//
// Where teacher and student nearly agree the loss is far smaller than the terms it is the sum of.  The exponentials of the
// classes outside the entries are float32: an error there changes the loss only in proportion to q_rest - p_rest.  They are
// added in float32 within a lane's pieces of a load (8 classes, 32 in rows that are streamed), beyond in float64, which the loads
// hide; rows of up to 128 classes, which the vector ALU bounds, take float32 throughout (8 classes a lane, then a tree).  What
// enters to first order (the entries' probabilities, the logarithms, the sum of the terms: K numbers per row) is float64.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace ocrhip {

namespace {

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const uint16_t* p) { return __uint_as_float((unsigned)*p << 16); }
__device__ __forceinline__ void store_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(uint16_t* p, float v) { *p = __builtin_bit_cast(uint16_t, (__bf16)v); }

// Order of the logits as unsigned integers: larger value, larger key; every NaN ranks above +infinity (below ~0, which no
// value has); -0 counts as 0.
__device__ __forceinline__ unsigned order_key(float x) {
    unsigned u = __float_as_uint(x + 0.0f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) u = 0x7FFFFFFEu;
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }

// ---- reductions over groups of 16, 32 or 64 lanes, on the vector ALU: quad, half row and row exchanges, then the swaps of
// rows and halves; every lane gets the same bits
template <int CTRL>
__device__ __forceinline__ unsigned lanes(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true); }
template <int CTRL>
__device__ __forceinline__ float lanes(float v) { return __uint_as_float(lanes<CTRL>(__float_as_uint(v))); }
template <int CTRL>
__device__ __forceinline__ double lanes(double v) {
    return __hiloint2double((int)lanes<CTRL>((unsigned)__double2hiint(v)), (int)lanes<CTRL>((unsigned)__double2loint(v)));
}
typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void rows16(unsigned v, unsigned& a, unsigned& b) {
    const uintx2 t = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    a = t[0]; b = t[1];
}
__device__ __forceinline__ void rows32(unsigned v, unsigned& a, unsigned& b) {
    const uintx2 t = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    a = t[0]; b = t[1];
}
template <bool HALF>
__device__ __forceinline__ void swapped(unsigned v, unsigned& a, unsigned& b) { HALF ? rows32(v, a, b) : rows16(v, a, b); }
template <bool HALF>
__device__ __forceinline__ void swapped(float v, float& a, float& b) {
    unsigned x, y;
    swapped<HALF>(__float_as_uint(v), x, y);
    a = __uint_as_float(x); b = __uint_as_float(y);
}
template <bool HALF>
__device__ __forceinline__ void swapped(double v, double& a, double& b) {
    unsigned xl, yl, xh, yh;
    swapped<HALF>((unsigned)__double2loint(v), xl, yl);
    swapped<HALF>((unsigned)__double2hiint(v), xh, yh);
    a = __hiloint2double((int)xh, (int)xl); b = __hiloint2double((int)yh, (int)yl);
}
template <int G, class T, class OP>
__device__ __forceinline__ T reduce(T v, OP op) {
    v = op(v, lanes<0xB1>(v));               // lane ^ 1
    v = op(v, lanes<0x4E>(v));               // lane ^ 2
    v = op(v, lanes<0x141>(v));              // the other quad of the half row
    v = op(v, lanes<0x140>(v));              // the other half row
    if (G >= 32) {
        T a, b;
        swapped<false>(v, a, b);
        v = op(a, b);
    }
    if (G == 64) {
        T a, b;
        swapped<true>(v, a, b);
        v = op(a, b);
    }
    return v;
}
template <int G, class T>
__device__ __forceinline__ T group_sum(T v) { return reduce<G>(v, [](T a, T b) { return a + b; }); }
template <int G>
__device__ __forceinline__ float group_max(float v) { return reduce<G>(v, [](float a, float b) { return fmaxf(a, b); }); }
template <int G>
__device__ __forceinline__ unsigned group_max(unsigned v) { return reduce<G>(v, [](unsigned a, unsigned b) { return a > b ? a : b; }); }
// the ballot of the lane's group
template <int G>
__device__ __forceinline__ unsigned long long group_ballot(bool b) {
    const unsigned long long w = __ballot(b);
    return G == 64 ? w : G == 32 ? w >> (threadIdx.x & 32) & 0xFFFFFFFFull : w >> (threadIdx.x & 48) & 0xFFFFull;
}

// ---- a row in pieces of 16 bytes, at any alignment of its elements
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_any __attribute__((ext_vector_type(8), aligned(2)));

template <class T>
constexpr int kPiece = 16 / sizeof(T);

// Piece q of a row of V classes, those from V on as -infinity.  The load has no branch - a load in one makes the compiler
// wait for the one in front of it -: the last piece is read from V - P on and put in place when it is used, pieces behind
// it are read like it.
__device__ __forceinline__ void unpack_piece(uintx4 t, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(t[i]);
}
__device__ __forceinline__ void unpack_piece(uintx4 t, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(t[i] << 16);
        v[2 * i + 1] = __uint_as_float(t[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ uintx4 pack_piece(const float (&v)[4]) {
    return uintx4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
__device__ __forceinline__ uintx4 pack_piece(const float (&v)[8]) {
    return __builtin_bit_cast(uintx4, bf16x8{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3], (__bf16)v[4], (__bf16)v[5], (__bf16)v[6], (__bf16)v[7]});
}
// TINY: rows shorter than a piece, element by element.
template <bool TINY, class T>
__device__ __forceinline__ uintx4 load_raw(const T* p, int q, int V) {
    constexpr int P = kPiece<T>;
    if constexpr (TINY) {
        float v[P];
#pragma unroll
        for (int e = 0; e < P; ++e) v[e] = load_f32(p + min(e, V - 1));
        return pack_piece(v);
    } else {
        return *reinterpret_cast<const uintx4_any*>(p + min(q * P, V - P));
    }
}
// t without its first 1, 2 or 4 classes, -infinity behind
template <int D>
__device__ __forceinline__ uintx4 drop(uintx4 t, const float*) {
    return D == 1 ? uintx4{t[1], t[2], t[3], 0xFF800000u} : uintx4{t[2], t[3], 0xFF800000u, 0xFF800000u};
}
template <int D>
__device__ __forceinline__ uintx4 drop(uintx4 t, const uint16_t*) {
    constexpr unsigned kNone = 0xFF80FF80u;
    if (D == 1) return uintx4{t[0] >> 16 | t[1] << 16, t[1] >> 16 | t[2] << 16, t[2] >> 16 | t[3] << 16, t[3] >> 16 | 0xFF800000u};
    return D == 2 ? uintx4{t[1], t[2], t[3], kNone} : uintx4{t[2], t[3], kNone, kNone};
}
template <bool TINY, class T>
__device__ __forceinline__ uintx4 in_place(uintx4 t, const T* p, int q, int V) {
    constexpr int P = kPiece<T>;
    if constexpr (TINY) {
        float v[P];
        unpack_piece(t, v);
#pragma unroll
        for (int e = 0; e < P; ++e) v[e] = q == 0 && e < V ? v[e] : -INFINITY;
        return pack_piece(v);
    }
    if ((q + 1) * P > V) {
        const int d = q * P - (V - P);
        if (d & 1) t = drop<1>(t, p);
        if (d & 2) t = drop<2>(t, p);
        if (P == 8 && d & 4) t = drop<4>(t, p);
        if (d >= P) {
            constexpr unsigned kNone = P == 8 ? 0xFF80FF80u : 0xFF800000u;
            t = uintx4{kNone, kNone, kNone, kNone};
        }
    }
    return t;
}
__device__ __forceinline__ void store_piece(float* p, int c, int V, const float* v) {
    if (c * 4 + 4 <= V) {
        *reinterpret_cast<floatx4_any*>(p + c * 4) = floatx4{v[0], v[1], v[2], v[3]};
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c * 4 + e < V) p[c * 4 + e] = v[e];
}
__device__ __forceinline__ void store_piece(uint16_t* p, int c, int V, const float* v) {
    if (c * 8 + 8 <= V) {
        *reinterpret_cast<bf16x8_any*>(p + c * 8) = bf16x8{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3], (__bf16)v[4], (__bf16)v[5], (__bf16)v[6], (__bf16)v[7]};
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (c * 8 + e < V) store_f32(p + c * 8 + e, v[e]);
}

constexpr float kLog2e = 1.44269504088896340736f;

// ---- float64 for a row's few numbers: each a fraction of the library's instructions, which a short row is bound by
//
// 1 / x, x neither 0 nor infinite: two Newton steps from the instruction's estimate.
__device__ __forceinline__ double rcp64(double x) {
    double r = __builtin_amdgcn_rcp(x);
    r = fma(fma(-x, r, 1.0), r, r);
    return fma(fma(-x, r, 1.0), r, r);
}
// exp(x): x = n ln 2 + r, |r| <= ln 2 / 2, the series of exp to r^12 / 12! (the next term is 2e-16 of the value); 0 from
// -infinity to -800, NaN stays NaN (and +infinity becomes one).  ln 2 is its first 40 bits behind the point, which n times are
// exact, and the rest.
__device__ __forceinline__ double exp64(double x) {
    x = x < -800.0 ? -800.0 : x;
    const double n = rint(x * 1.4426950408889634074);
    const double r = fma(n, 1.7239444525614835e-13, fma(n, -0.6931471805601177, x));
    double p = 1.0 / 479001600.0;
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return __builtin_amdgcn_ldexp(p, (int)n);
}
// log(x), x positive and finite: x = 2^e m, sqrt(1/2) <= m < sqrt(2), s = (m - 1) / (m + 1), |s| < 0.172, log m =
// 2 (s + s^3 / 3 + ... + s^21 / 21).  NaN stays NaN.
__device__ __forceinline__ double log64(double x) {
    double m = __builtin_amdgcn_frexp_mant(x);
    int e = __builtin_amdgcn_frexp_exp(x);
    const bool low = m < 0.70710678118654752440;
    m = low ? m + m : m;
    e = low ? e - 1 : e;
    const double s = (m - 1.0) * rcp64(m + 1.0), q = s * s;
    double p = 2.0 / 21.0;
    p = fma(p, q, 2.0 / 19.0);
    p = fma(p, q, 2.0 / 17.0);
    p = fma(p, q, 2.0 / 15.0);
    p = fma(p, q, 2.0 / 13.0);
    p = fma(p, q, 2.0 / 11.0);
    p = fma(p, q, 2.0 / 9.0);
    p = fma(p, q, 2.0 / 7.0);
    p = fma(p, q, 2.0 / 5.0);
    p = fma(p, q, 2.0 / 3.0);
    return fma((double)e, 0.69314718055994530942, fma(p * q, s, 2.0 * s));
}
// log of a sum of exponentials, which may be 0 or infinite
__device__ __forceinline__ double log_sum(double x) { return x == 0.0 ? -INFINITY : x == INFINITY ? x : log64(x); }

constexpr int kShort = 128;            // classes of a row that 16 lanes share

// what one lane wrote to LDS is what another reads: same wave, so the order of the instructions is enough
__device__ __forceinline__ void lds_phase() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

// ---- top logits
//
// Bound by reading the logits once.  Rows of up to 128 classes: 16 lanes per row (top16_kernel).  Longer rows:
// the K-th largest of the lanes' own maxima is a lower bound of the K-th largest of all (K lanes hold a value that large),
// and hardly more than K values reach it: it is found by bisection of its leading bits, the values that reach it are put on
// a list in LDS and each finds its rank by counting the larger ones.  A row with too many candidates (hundreds of equal
// values, as under a mask) takes the few above the K-th largest and the first of those equal to it, or failing that its
// maxima one by one.
template <class T>
struct TopArgs {
    const T* x;
    int64_t ld, rows;
    int V, K;
    float inv_t;
    float* values;
    int* index;
    float* lse;
};

// Every lane sorts its 8 classes, the lists go to LDS, and the K largest of the row are K times the largest head of 16 lists;
// the winner writes its class down and moves on.  Bound by the vector ALU (1.4M rows of 97 float32, 10 entries: 328 us, 1.7
// TB/s): the next row's loads are on their way, and a logit's key with its class (7 bits; among equals the lower class counts
// as the larger) is held as the bits of a float64 between 1 and 2, which order like the numbers: two instructions sort a
// pair.
__device__ __forceinline__ double entry_of(unsigned key, unsigned at) {
    return __hiloint2double((int)(0x3FF00000u | key >> 12), (int)(key << 20 | (127u - at) << 13));
}
__device__ __forceinline__ unsigned entry_key(unsigned hi, unsigned lo) { return hi << 12 | lo >> 20; }
__device__ __forceinline__ unsigned entry_class(unsigned lo) { return 127u - (lo >> 13 & 127u); }

template <class T, bool TINY>
__global__ __launch_bounds__(256) void top16_kernel(TopArgs<T> a) {
    constexpr int P = kPiece<T>, L = kShort / 16, N = L / P;
    __shared__ double lists[L][256];                       // from the third on; two entries below all behind the last
    extern __shared__ double found_lds[];                  // K per row
    const int tid = threadIdx.x, part = tid & 15, sub = tid >> 4;
    double* found = found_lds + sub * a.K;
    const float c = a.inv_t * kLog2e;
    const int64_t step = (int64_t)gridDim.x * 16;
    uintx4 next[N];
    auto fetch = [&](int64_t row) {
        const T* p = a.x + min(row, a.rows - 1) * a.ld;
#pragma unroll
        for (int i = 0; i < N; ++i) next[i] = load_raw<TINY>(p, part + 16 * i, a.V);
    };
    int64_t row = (int64_t)blockIdx.x * 16 + sub;
    fetch(row);
    lists[L - 2][tid] = 1.0;
    lists[L - 1][tid] = 1.0;
    for (int64_t first_row = (int64_t)blockIdx.x * 16; first_row < a.rows; first_row += step, row += step) {
        float v[L];
        double own[L];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float w[P];
            unpack_piece(in_place<TINY>(next[i], a.x, part + 16 * i, a.V), w);
#pragma unroll
            for (int e = 0; e < P; ++e) {
                const unsigned at = (unsigned)((part + 16 * i) * P + e);
                v[i * P + e] = w[e];
                own[i * P + e] = at < (unsigned)a.V ? entry_of(order_key(w[e]), at) : 1.0;
            }
        }
        fetch(row + step);
        constexpr int order[19][2] = {{0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6}, {5, 7}, {1, 2}, {5, 6},
                                      {0, 4}, {1, 5}, {2, 6}, {3, 7}, {2, 4}, {3, 5}, {1, 2}, {3, 4}, {5, 6}};
#pragma unroll
        for (int i = 0; i < 19; ++i) {
            const double x = own[order[i][0]], y = own[order[i][1]];
            own[order[i][0]] = __builtin_fmax(x, y);
            own[order[i][1]] = __builtin_fmin(x, y);
        }
#pragma unroll
        for (int i = 2; i < L; ++i) lists[i - 2][tid] = own[i];
        unsigned hi = (unsigned)__double2hiint(own[0]), lo = (unsigned)__double2loint(own[0]);
        double second = own[1];
        const double* behind = &lists[0][tid];
        for (int k = 0; k < a.K; ++k) {                    // K <= V: some head is a class
            const unsigned top = group_max<16>(hi), which = group_max<16>(hi == top ? lo : 0u);
            if (hi == top && lo == which) {
                found[k] = __hiloint2double((int)hi, (int)lo);
                hi = (unsigned)__double2hiint(second);
                lo = (unsigned)__double2loint(second);
                second = *behind;
                behind += 256;
            }
        }
        lds_phase();
        if (a.lse) {
            const float high = key_value(entry_key((unsigned)__double2hiint(found[0]), (unsigned)__double2loint(found[0])));
            const float base = fabsf(high) == INFINITY || high != high ? 0.0f : high;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < L; ++i) sum += __builtin_amdgcn_exp2f((v[i] - base) * c);
            sum = group_sum<16>(sum);
            if (part == 0 && row < a.rows) a.lse[row] = (float)((double)base * a.inv_t + log_sum((double)sum));
        }
        if (row < a.rows)
            for (int k = part; k < a.K; k += 16) {
                const unsigned h = (unsigned)__double2hiint(found[k]), l = (unsigned)__double2loint(found[k]);
                a.values[row * a.K + k] = key_value(entry_key(h, l));
                a.index[row * a.K + k] = (int)entry_class(l);
            }
        lds_phase();
    }
}

// Rows in LDS: short ones are one wave's own, so that nothing waits for another; longer ones are shared, for few fit a compute
// unit (which waves take which rows: launch_top, launch_distill).
constexpr size_t kWaveBytes = 16384, kRowBytes = 32768;
constexpr int kTopList = 512;          // candidates of a row that LDS holds

// The row to LDS, BATCH pieces of a lane in flight (pieces of 16 bytes; classes behind the last are -infinity); returns the
// lane's maximum.  `between` runs while the first pieces are on their way.
template <int THREADS, int BATCH, bool TINY, class T, class F>
__device__ __forceinline__ float row_to_lds(const T* p, int V, uintx4* buf, F between) {
    constexpr int P = kPiece<T>;
    const int pieces = (V + P - 1) / P, tid = threadIdx.x;
    float m = -INFINITY;
    for (int q = tid; q - tid < pieces; q += THREADS * BATCH) {
        uintx4 t[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
            t[i] = load_raw<TINY>(p, q + i * THREADS, V);
        if (q == tid) between();
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
            if (q + i * THREADS < pieces) {
                const uintx4 u = in_place<TINY>(t[i], p, q + i * THREADS, V);
                float v[P];
                unpack_piece(u, v);
#pragma unroll
                for (int e = 0; e < P; ++e) m = fmaxf(m, v[e]);
                buf[q + i * THREADS] = u;
            }
    }
    return m;
}

// the largest bound that K of the wave's keys reach (0: fewer than K lanes have one), its bits from FROM down to TO; those in
// front of them are given
template <int FROM, int TO>
__device__ __forceinline__ unsigned bisect(const unsigned* keys, int n, int K, unsigned bound = 0) {
    for (int bit = FROM; bit >= TO; --bit) {
        const unsigned next = bound | 1u << bit;
        int reach = 0;
        for (int w = 0; w < n; ++w) reach += __popcll(__ballot(keys[w] >= next));
        if (reach >= K) bound = next;
    }
    return bound;
}

// The K largest of the list, each at the rank that counting the larger ones gives it.
template <class T>
__device__ __forceinline__ void write_ranked(const TopArgs<T>& a, int64_t row, const unsigned long long* list, int n, int tid, int threads) {
    for (int i = tid; i < n; i += threads) {
        const unsigned long long own = list[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += list[j] > own ? 1 : 0;
        if (rank < a.K) {
            a.values[row * a.K + rank] = key_value((unsigned)(own >> 32));
            a.index[row * a.K + rank] = (int)(0xFFFFFFFFu - (unsigned)own);
        }
    }
}

// The same for a row that has more candidates than the list holds, with a key that at least K values reach.  Mostly the K-th
// largest value is that key and many others are equal to it (classes masked with one low value, a row without a finite
// logit): the fewer than K values above it go to the list, then the first equal ones in the order of the classes.  False
// where K values or more lie above it.
template <int WAVES, class T>
__device__ __forceinline__ bool write_equal(const TopArgs<T>& a, int64_t row, unsigned key, unsigned long long* list, int* count) {
    const int tid = threadIdx.x, lane = tid & 63;
    const T* p = a.x + row * a.ld;
    __syncthreads();                                       // every thread has read the count that led here
    if (tid == 0) *count = 0;
    __syncthreads();
    for (int at = tid; at < a.V; at += WAVES * 64) {
        const unsigned own = order_key(load_f32(p + at));
        if (own > key) {
            const int slot = atomicAdd(count, 1);
            if (slot < a.K) list[slot] = (unsigned long long)own << 32 | (0xFFFFFFFFu - (unsigned)at);
        }
    }
    __syncthreads();
    const int above = *count;
    if (above >= a.K) return false;
    if (tid < 64) {
        int have = above;
        for (int base = 0; base < a.V && have < a.K; base += 64) {
            const int at = base + lane;
            const bool equal = at < a.V && order_key(load_f32(p + min(at, a.V - 1))) == key;
            const unsigned long long all = __ballot(equal);
            const int slot = have + __popcll(all & ((1ull << lane) - 1));
            if (equal && slot < a.K) list[slot] = (unsigned long long)key << 32 | (0xFFFFFFFFu - (unsigned)at);
            have += __popcll(all);
        }
    }
    __syncthreads();
    write_ranked(a, row, list, a.K, tid, WAVES * 64);
    return true;
}

// The same without a list: the maxima one by one, a pass over the row each.
template <int WAVES, class T>
__device__ __forceinline__ void write_one_by_one(const TopArgs<T>& a, int64_t row, unsigned long long* wave_best) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T* p = a.x + row * a.ld;
    unsigned long long last = ~0ull;
    for (int k = 0; k < a.K; ++k) {
        unsigned long long best = 0;
        for (int at = tid; at < a.V; at += WAVES * 64) {
            const unsigned long long own = (unsigned long long)order_key(load_f32(p + at)) << 32 | (0xFFFFFFFFu - (unsigned)at);
            if (own < last && own > best) best = own;
        }
        const unsigned hi = group_max<64>((unsigned)(best >> 32));
        const unsigned lo = group_max<64>((unsigned)(best >> 32) == hi ? (unsigned)best : 0u);
        if (lane == 0) wave_best[wave] = (unsigned long long)hi << 32 | lo;
        __syncthreads();
        last = wave_best[0];
        for (int w = 1; w < WAVES; ++w) last = max(last, wave_best[w]);
        __syncthreads();
        if (tid == 0) {
            a.values[row * a.K + k] = key_value((unsigned)(last >> 32));
            a.index[row * a.K + k] = (int)(0xFFFFFFFFu - (unsigned)last);
        }
    }
}

// A row in LDS, W waves on it (FEW: as many maxima a lane as a piece has classes, one wave): bound by reading the logits (16384
// rows of 6719 float32, 32 entries: 98 us, 4.5 TB/s).  The bound of the candidates: every wave bisects its own 64 maxima for
// the ceil(K / W)-th largest, the least of those is reached by at least K values.
template <class T, int W, int BATCH, bool FEW = false>
__global__ __launch_bounds__(W * 64) void top_lds_kernel(TopArgs<T> a) {
    constexpr int P = kPiece<T>, THREADS = W * 64;
    extern __shared__ uintx4 buf[];                        // the row
    __shared__ unsigned long long list[kTopList], wave_best[W];
    __shared__ unsigned wave_bits[W];
    __shared__ float wave_top[W];
    __shared__ double wave_sum[W];
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, pieces = (a.V + P - 1) / P;
    const float c = a.inv_t * kLog2e;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        if (tid == 0) count = 0;
        const float mine = row_to_lds<THREADS, BATCH, false>(a.x + row * a.ld, a.V, buf, [] {});
        const unsigned key = tid < pieces ? order_key(mine) : 0u;
        unsigned fine[P] = {};
        if (FEW) {
            float part[P];
#pragma unroll
            for (int e = 0; e < P; ++e) part[e] = -INFINITY;
            lds_phase();
            for (int q = tid; q < pieces; q += THREADS) {
                float v[P];
                unpack_piece(buf[q], v);
#pragma unroll
                for (int e = 0; e < P; ++e) part[e] = fmaxf(part[e], v[e]);
            }
#pragma unroll
            for (int e = 0; e < P; ++e) fine[e] = tid * P + e < a.V ? order_key(part[e]) : 0u;
        }
        const unsigned own_least = FEW ? bisect<31, 12>(fine, P, a.K) : bisect<31, 12>(&key, 1, (a.K + W - 1) / W);
        unsigned least = own_least;
        float high = group_max<64>(mine);                  // NaN apart
        if (W > 1) {
            if (lane == 0) {
                wave_bits[wave] = least;
                wave_top[wave] = high;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < W; ++i) {
                least = min(least, wave_bits[i]);
                high = fmaxf(high, wave_top[i]);
            }
        }
        lds_phase();
        const float bound = least ? key_value(least) : -INFINITY;
        const float base = fabsf(high) == INFINITY ? 0.0f : high;
        double sum = 0.0;
        for (int q = tid; q < pieces; q += THREADS) {      // its own pieces
            float v[P], part = 0.0f;
            unpack_piece(buf[q], v);
            bool any = false;
#pragma unroll
            for (int e = 0; e < P; ++e) {
                any |= !(v[e] < bound);                    // a NaN as well
                part += __builtin_amdgcn_exp2f((v[e] - base) * c);
            }
            sum += (double)part;
            if (any)
#pragma unroll
                for (int e = 0; e < P; ++e)
                    if (!(v[e] < bound) && q * P + e < a.V) {
                        const int slot = atomicAdd(&count, 1);
                        if (slot < kTopList) list[slot] = (unsigned long long)order_key(v[e]) << 32 | (0xFFFFFFFFu - (unsigned)(q * P + e));
                    }
        }
        sum = group_sum<64>(sum);
        if (lane == 0) wave_sum[wave] = sum;
        __syncthreads();
        const int n = count;
        if (a.lse && tid == THREADS - 1) {
            double total = 0.0;
            for (int i = 0; i < W; ++i) total += wave_sum[i];
            a.lse[row] = (float)((double)base * a.inv_t + log_sum(total));
        }
        if (n <= kTopList) {
            write_ranked(a, row, list, n, tid, THREADS);
        } else {
            unsigned exact = FEW ? bisect<11, 0>(fine, P, a.K, own_least) : bisect<11, 0>(&key, 1, (a.K + W - 1) / W, own_least);
            if (W > 1) {
                if (lane == 0) wave_bits[wave] = exact;
                __syncthreads();
                exact = wave_bits[0];
#pragma unroll
                for (int i = 1; i < W; ++i) exact = min(exact, wave_bits[i]);
            }
            if (!write_equal<W>(a, row, exact, list, &count)) write_one_by_one<W>(a, row, wave_best);
        }
        __syncthreads();
    }
}

// Longer rows: 8 waves per row, which is read twice, for the threads' maxima (and the sum) and for the values that reach
// the bound.
template <class T>
__global__ __launch_bounds__(512) void top_stream_kernel(TopArgs<T> a) {
    constexpr int P = kPiece<T>, WAVES = 8, THREADS = 512, AHEAD = 4;
    __shared__ unsigned long long list[kTopList];
    __shared__ unsigned maxima[THREADS];
    __shared__ double wave_sum[WAVES];
    __shared__ unsigned long long wave_best[WAVES];
    __shared__ unsigned shared_bound, shared_exact;
    __shared__ float shared_high;
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int pieces = (a.V + P - 1) / P;
    const float c = a.inv_t * kLog2e;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* p = a.x + row * a.ld;
        float m_own = -INFINITY;                           // running maximum and sum of the thread
        double s_own = 0.0;
        if (tid == 0) count = 0;
        for (int q = tid; q < pieces; q += THREADS * AHEAD) {
            uintx4 raw[AHEAD];
            float w[AHEAD][P];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) raw[i] = load_raw<false>(p, q + i * THREADS, a.V);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) unpack_piece(in_place<false>(raw[i], p, q + i * THREADS, a.V), w[i]);
            float m = m_own;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
#pragma unroll
                for (int e = 0; e < P; ++e) m = fmaxf(m, w[i][e]);
            const float base = fabsf(m) == INFINITY ? 0.0f : m;
            s_own = fabsf(m_own) == INFINITY ? s_own : s_own * (double)__builtin_amdgcn_exp2f((m_own - base) * c);
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
#pragma unroll
                for (int e = 0; e < P; ++e) part += __builtin_amdgcn_exp2f((w[i][e] - base) * c);
            s_own += (double)part;
            m_own = m;
        }
        maxima[tid] = tid < pieces ? order_key(m_own) : 0u;
        __syncthreads();
        if (wave == 0) {
            unsigned m[WAVES], top = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                m[w] = maxima[w * 64 + lane];
                top = max(top, m[w]);
            }
            const unsigned bits = bisect<31, 12>(m, WAVES, a.K);
            top = group_max<64>(top);
            if (lane == 0) {
                shared_bound = bits;
                shared_high = key_value(top);
            }
        }
        __syncthreads();
        const float bound = shared_bound ? key_value(shared_bound) : -INFINITY;
        const float high = shared_high, base = fabsf(high) == INFINITY ? 0.0f : high;
        // a thread whose values all lie below the bound has nothing to offer (one that met a NaN has it in its sum)
        if (!(m_own < bound) || s_own != s_own)
            for (int q = tid; q < pieces; q += THREADS) {
                float v[P];
                unpack_piece(in_place<false>(load_raw<false>(p, q, a.V), p, q, a.V), v);
#pragma unroll
                for (int e = 0; e < P; ++e)
                    if (!(v[e] < bound) && q * P + e < a.V) {
                        const int slot = atomicAdd(&count, 1);
                        if (slot < kTopList) list[slot] = (unsigned long long)order_key(v[e]) << 32 | (0xFFFFFFFFu - (unsigned)(q * P + e));
                    }
            }
        const float own_base = fabsf(m_own) == INFINITY ? 0.0f : m_own;
        const double sum = group_sum<64>(m_own == -INFINITY ? s_own : s_own * (double)__builtin_amdgcn_exp2f((own_base - base) * c));
        if (lane == 0) wave_sum[wave] = sum;
        __syncthreads();
        const int n = count;
        if (n <= kTopList) {
            write_ranked(a, row, list, n, tid, THREADS);
        } else {
            if (wave == 0) {
                unsigned m[WAVES];
#pragma unroll
                for (int w = 0; w < WAVES; ++w) m[w] = maxima[w * 64 + lane];
                const unsigned exact = bisect<11, 0>(m, WAVES, a.K, shared_bound);
                if (lane == 0) shared_exact = exact;
            }
            __syncthreads();
            if (!write_equal<WAVES>(a, row, shared_exact, list, &count)) write_one_by_one<WAVES>(a, row, wave_best);
        }
        if (a.lse && tid == 0) {
            double total = 0.0;
            for (int w = 0; w < WAVES; ++w) total += wave_sum[w];
            a.lse[row] = (float)((double)base * a.inv_t + log_sum(total));
        }
        __syncthreads();
    }
}

// ---- distillation

// A group of G lanes (16, 32 or 64, K <= G), lane k = entry k; float64 throughout.
//
// With d_k = (s_k - m) / tau, S = sum of exp((s - m) / tau) over all classes and S_r over those outside the entries, so that
// log q_k = d_k - log S and log q_rest = log S_r - log S:
//   loss = sum p_k (log p_k - d_k) + p_rest (log(p_rest / S_r)) + (sum p_k + p_rest) log S
// and without the rest, log p_k = z_k / tau - top - log E, E = sum of exp(z / tau - top), sum p_k = 1:
//   loss = sum p_k (z_k / tau - top - d_k) + log(S / E).
struct Teacher {        // what the teacher's entries alone make of a row
    double p, log_p;    // of the lane's entry; without the rest log_p lacks - log E
    double mass;        // sum of the p_k
    double rest;        // p_rest, or 1 / E without the rest
    bool any;           // there is some probability (always with the log normaliser)
};
template <int G>
__device__ __forceinline__ Teacher teacher_of(bool there, float z, bool has_lse, float lse, double inv_t) {
    Teacher o;
    o.any = true;
    if (has_lse) {
        o.log_p = there && z != -INFINITY ? fma((double)z, inv_t, -(double)lse) : -INFINITY;       // lse may be -infinity too
        o.p = exp64(o.log_p);
        o.mass = group_sum<G>(o.p);
        o.rest = o.mass >= 1.0 ? 0.0 : 1.0 - o.mass;
    } else {
        const float top = group_max<G>(there ? z : -INFINITY);
        o.any = top != -INFINITY || group_ballot<G>(there && z != z) != 0;
        o.log_p = there ? ((double)z - top) * inv_t : -INFINITY;
        const double e = exp64(o.log_p);
        o.rest = rcp64(group_sum<G>(e));
        o.p = e * o.rest;
        o.mass = 1.0;
    }
    return o;
}

// The row: the entries' logits s_k and, of the classes outside the entries, a base m_r and sum_r = sum of
// exp((s - m_r) / tau).  m_r -infinity: nothing finite there.
struct RowResult {
    double loss;        // without weight and tau^2
    double coef;        // gradient of a class outside the entries = coef * exp((s - m_r) / tau)
    double grad_k;      // gradient of the lane's class (where the lane is its first entry)
    bool first;         // the lane's entry is there and no lower lane names its class
};
template <int G>
__device__ __forceinline__ RowResult row_result(const Teacher& t, int K, bool there, bool again, int idx, float s_k, bool has_lse, double inv_t, float m_r,
                                                double sum_r, int V) {
    RowResult out;
    const int lane = threadIdx.x & (G - 1);
    bool first = there;
    const bool doubled = group_ballot<G>(again) != 0;          // some class is named twice
    if (doubled)
        for (int j = 0; j < K; ++j) {
            const int other = __shfl(there ? idx : -1, j, G);
            if (j < lane && there && other == idx) first = false;
        }
    const float m = fmaxf(m_r, group_max<G>(first ? s_k : -INFINITY));
    const double d_k = ((double)s_k - m) * inv_t, d_r = ((double)m_r - m) * inv_t;
    const double e_k = first ? exp64(d_k) : 0.0;
    double shift = m_r == -INFINITY ? 0.0 : 1.0;
    if (m_r != m && m_r != -INFINITY) shift = exp64(d_r);
    const double total = group_sum<G>(e_k) + sum_r * shift, inv_total = rcp64(total);
    double sum_same = t.p, p_k = t.p, log_p = t.log_p;
    if (doubled) {                                             // entries of one class add up, in its first lane
        sum_same = 0.0;
        for (int j = 0; j < K; ++j) {
            const int other = __shfl(there ? idx : -1, j, G);
            const double pj = __shfl(t.p, j, G);
            if (there && other == idx) sum_same += pj;
        }
        p_k = first ? sum_same : 0.0;
        if (first && sum_same != t.p) log_p = log64(sum_same) - (has_lse ? 0.0 : log64(t.rest));
    }
    double loss = group_sum<G>(p_k == 0.0 ? 0.0 : p_k * (log_p - d_k));
    double of_q = inv_total, coef = shift * inv_total;
    if (has_lse) {
        const bool rest = t.rest != 0.0 && __popcll(group_ballot<G>(first)) != V;
        const double all = t.mass + (rest ? t.rest : 0.0);
        loss += all * log64(total);
        of_q *= all;
        coef *= all;
        if (rest && m_r == -INFINITY)
            loss += INFINITY;                              // a NaN of the entries stays one
        else if (rest) {
            const double ratio = t.rest * rcp64(sum_r);
            loss += t.rest * (log64(ratio) - d_r);
            coef -= ratio;
        }
    } else {
        loss += log64(total * t.rest);
    }
    out.first = first;
    out.loss = t.any ? loss : 0.0;
    out.coef = !t.any ? 0.0 : loss != loss ? loss : coef;
    out.grad_k = !t.any ? 0.0 : loss != loss ? loss : e_k * of_q - sum_same;
    return out;
}

template <class T>
struct DistillArgs {
    const T* x;
    int64_t ld, ld_grad, rows;
    const float *values, *lse, *weight;
    const int* index;
    float* loss;
    T* grad;
    int V, K;
    float t;
};

// What the entries do to a row in LDS, a group of lanes, lane k = entry k: returns its class's logit and leaves -infinity in
// its place.  `again`: the lane's class is named by another lane too, whose mark stayed.
template <class T>
__device__ __forceinline__ float take_entry(void* row, bool there, int idx, int lane, bool& again) {
    typedef T __attribute__((may_alias)) slot_t;
    typedef __attribute__((may_alias)) typename std::conditional<sizeof(T) == 4, unsigned, uint16_t>::type mark_t;
    mark_t* marks = reinterpret_cast<mark_t*>(row);
    const float s_k = there ? load_f32(reinterpret_cast<const T*>(reinterpret_cast<slot_t*>(row) + idx)) : -INFINITY;
    lds_phase();
    if (there) marks[idx] = (mark_t)lane;
    lds_phase();
    again = there && (int)marks[idx] != lane;
    lds_phase();
    if (there) marks[idx] = sizeof(T) == 4 ? (mark_t)0xFF800000u : (mark_t)0xFF80u;
    lds_phase();
    return s_k;
}
template <class T>
__device__ __forceinline__ void put_entry(void* row, int idx, float v) {
    typedef T __attribute__((may_alias)) slot_t;
    store_f32(reinterpret_cast<T*>(reinterpret_cast<slot_t*>(row) + idx), v);
}

// Rows of up to 128 classes: as many lanes per row as it has entries, at least 16, in LDS of the group's own.  Such a row is 776
// bytes and a few hundred float64 instructions (131072 rows of 97 float32, 10 entries: 31 us, 3.7 TB/s, bound by the vector
// ALU), so the next row's loads (and the weight of the one after it, which says whether to load it) are on their way while
// one is worked on.
template <class T, bool TINY, int G>
__global__ __launch_bounds__(256) void distill_short_kernel(DistillArgs<T> a) {
    constexpr int ROWS = 256 / G, P = kPiece<T>, N = kShort / P > G ? kShort / P / G : 1;
    __shared__ uintx4 rows_lds[ROWS][N * G];
    const int part = threadIdx.x & (G - 1), sub = threadIdx.x / G, pieces = (a.V + P - 1) / P;
    uintx4* buf = rows_lds[sub];
    const double inv_t = 1.0 / a.t;
    const float c = kLog2e / a.t;
    const int64_t step = (int64_t)gridDim.x * ROWS;
    auto weight_of = [&](int64_t row) { return row >= a.rows ? 0.0f : a.weight ? a.weight[row] : 1.0f; };
    uintx4 next[N];
    int next_idx;
    float next_z, next_lse = 0.0f;
    auto fetch = [&](int64_t row, bool live) {                 // no branch: a row that is not wanted loads the first one
        const int64_t r = live ? row : 0;
        const T* p = a.x + r * a.ld;
#pragma unroll
        for (int i = 0; i < N; ++i) next[i] = load_raw<TINY>(p, part + i * G, a.V);
        const int64_t k = r * a.K + min(part, a.K - 1);
        next_idx = a.index[k];
        next_z = a.values[k];
        if (a.lse) next_lse = a.lse[r];
    };
    int64_t row = (int64_t)blockIdx.x * ROWS + sub;
    float w_next = weight_of(row);
    fetch(row, w_next != 0.0f);
    float w_after = weight_of(row + step);
    for (int64_t first_row = (int64_t)blockIdx.x * ROWS; first_row < a.rows; first_row += step, row += step) {
        const float w = w_next;
        const bool in_range = row < a.rows, live = w != 0.0f;  // lanes without a row run along
        const int idx = live && part < a.K ? next_idx : -1;
        const float z = next_z, lse = next_lse;
        const bool there = idx >= 0 && idx < a.V;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float v[P];
            const uintx4 u = in_place<TINY>(next[i], a.x, part + i * G, a.V);
            unpack_piece(u, v);
#pragma unroll
            for (int e = 0; e < P; ++e) top = fmaxf(top, v[e]);
            buf[part + i * G] = u;
        }
        w_next = w_after;
        fetch(row + step, w_next != 0.0f);
        w_after = weight_of(row + 2 * step);
        lds_phase();
        bool again;
        const float s_k = take_entry<T>(buf, there, idx, part, again);
        float v[N][P], m_r = group_max<G>(top);
        auto sum_of = [&](float base) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                unpack_piece(buf[part + i * G], v[i]);
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    v[i][e] = __builtin_amdgcn_exp2f((v[i][e] - base) * c);
                    sum += v[i][e];
                }
            }
            return group_sum<G>(sum);
        };
        float sum_r = sum_of(m_r == -INFINITY ? 0.0f : m_r);
        if (__ballot(sum_r < 1e-20f)) {      // some row of the wave: far below its entries, so from its own maximum
            float own = -INFINITY;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float u[P];
                unpack_piece(buf[part + i * G], u);
#pragma unroll
                for (int e = 0; e < P; ++e) own = fmaxf(own, u[e]);
            }
            own = group_max<G>(own);
            m_r = sum_r < 1e-20f ? own : m_r;
            sum_r = sum_of(m_r == -INFINITY ? 0.0f : m_r);
        }
        const Teacher t = teacher_of<G>(there, z, a.lse != nullptr, lse, inv_t);
        // a NaN outside the entries: the maximum does not see it, the sum does
        const RowResult r = row_result<G>(t, a.K, there, again, idx, s_k, a.lse != nullptr, inv_t, sum_r != sum_r ? NAN : m_r, (double)sum_r, a.V);
        const double scale = (double)w * a.t;
        if (a.loss && in_range && part == 0) a.loss[row] = live ? (float)(r.loss * scale * a.t) : 0.0f;
        if (a.grad) {
            const float coef = live ? (float)(r.coef * scale) : 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
#pragma unroll
                for (int e = 0; e < P; ++e) v[i][e] = coef != 0.0f ? coef * v[i][e] : 0.0f;
                buf[part + i * G] = pack_piece(v[i]);
            }
            lds_phase();
            if (r.first) put_entry<T>(buf, idx, (float)(r.grad_k * scale));
            lds_phase();
            T* g = a.grad + row * a.ld_grad;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                unpack_piece(buf[part + i * G], v[i]);
                if (in_range && part + i * G < pieces) store_piece(g, part + i * G, a.V, v[i]);
            }
        }
        lds_phase();
    }
}

// A row in LDS, W waves on it: read from memory once, bound by that and by writing the gradient (16384 rows of 6719 bfloat16
// 101 us, 4.4 TB/s).  The first wave has the entries, and does the teacher's part while
// the row is on its way.  The entries' places hold -infinity during the sum, so that nothing has to be tested per class;
// every wave turns its own pieces into gradients in place, puts the entries' gradients among them and stores whole pieces.
template <class T, int W, int BATCH, bool TINY>
__global__ __launch_bounds__(W * 64) void distill_lds_kernel(DistillArgs<T> a) {
    constexpr int P = kPiece<T>, THREADS = W * 64;
    extern __shared__ uintx4 buf[];
    __shared__ double wave_sum[W];
    __shared__ float wave_top[W], entry_grad[64];
    __shared__ int entry_class[64];
    __shared__ float shared_coef;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, pieces = (a.V + P - 1) / P;
    const double inv_t = 1.0 / a.t;
    const float c = kLog2e / a.t;
    auto over_waves = [&](auto* part, auto v, auto op) {                 // of the waves' values, in their order
        if (W == 1) return v;
        if (lane == 0) part[wave] = v;
        __syncthreads();
        auto o = part[0];
#pragma unroll
        for (int i = 1; i < W; ++i) o = op(o, part[i]);
        return o;
    };
    auto larger = [](float a, float b) { return fmaxf(a, b); };
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        T* g = a.grad ? a.grad + row * a.ld_grad : nullptr;
        const float w = a.weight ? a.weight[row] : 1.0f;
        if (w == 0.0f) {
            if (tid == 0 && a.loss) a.loss[row] = 0.0f;
            float zeros[P] = {};
            if (g)
                for (int q = tid; q < pieces; q += THREADS) store_piece(g, q, a.V, zeros);
            continue;
        }
        int idx = -1;
        float z = 0.0f;
        if (wave == 0 && lane < a.K) {
            idx = a.index[row * a.K + lane];
            z = a.values[row * a.K + lane];
        }
        const float lse = a.lse ? a.lse[row] : 0.0f;
        const bool there = idx >= 0 && idx < a.V;
        Teacher t;
        const float own_top = row_to_lds<THREADS, BATCH, TINY>(a.x + row * a.ld, a.V, buf, [&] {
            if (wave == 0) t = teacher_of<64>(there, z, a.lse != nullptr, lse, inv_t);
        });
        float m_r = over_waves(wave_top, group_max<64>(own_top), larger);
        if (W == 1) lds_phase();
        float s_k = -INFINITY;
        bool again = false;
        if (wave == 0) s_k = take_entry<T>(buf, there, idx, lane, again);
        if (W > 1) __syncthreads();
        auto sum_of = [&](float base) {
            double sum = 0.0;
            for (int q = tid; q < pieces; q += THREADS) {
                float v[P], part = 0.0f;
                unpack_piece(buf[q], v);
#pragma unroll
                for (int e = 0; e < P; ++e) part += __builtin_amdgcn_exp2f((v[e] - base) * c);
                sum += (double)part;
            }
            return over_waves(wave_sum, group_sum<64>(sum), [](double a, double b) { return a + b; });
        };
        float base = m_r == -INFINITY ? 0.0f : m_r;
        double sum_r = sum_of(base);
        if (sum_r < 1e-20) {               // far below the entries: from their own maximum
            m_r = -INFINITY;
            for (int q = tid; q < pieces; q += THREADS) {
                float v[P];
                unpack_piece(buf[q], v);
#pragma unroll
                for (int e = 0; e < P; ++e) m_r = fmaxf(m_r, v[e]);
            }
            m_r = over_waves(wave_top, group_max<64>(m_r), larger);
            base = m_r == -INFINITY ? 0.0f : m_r;
            sum_r = sum_of(base);
        }
        if (wave == 0) {
            // a NaN outside the entries: the maximum does not see it, the sum does
            const RowResult r = row_result<64>(t, a.K, there, again, idx, s_k, a.lse != nullptr, inv_t, sum_r != sum_r ? NAN : m_r, sum_r, a.V);
            const double scale = (double)w * a.t;
            if (lane == 0) {
                if (a.loss) a.loss[row] = (float)(r.loss * scale * a.t);
                shared_coef = (float)(r.coef * scale);
            }
            entry_class[lane] = r.first ? idx : -1;
            entry_grad[lane] = (float)(r.grad_k * scale);
        }
        if (W > 1) __syncthreads();
        if (W == 1) lds_phase();
        if (g) {
            const float coef = shared_coef;
            for (int q = tid; q < pieces; q += THREADS) {
                float v[P];
                unpack_piece(buf[q], v);
#pragma unroll
                for (int e = 0; e < P; ++e) v[e] = coef != 0.0f ? coef * __builtin_amdgcn_exp2f((v[e] - base) * c) : 0.0f;
                buf[q] = pack_piece(v);
            }
            lds_phase();
            const int mine = entry_class[lane];
            if (mine >= 0 && mine / P % THREADS / 64 == wave) put_entry<T>(buf, mine, entry_grad[lane]);
            lds_phase();
            for (int q = tid; q < pieces; q += THREADS) {
                const uintx4 t4 = buf[q];
                if ((q + 1) * P <= a.V) {
                    *reinterpret_cast<uintx4_any*>(g + q * P) = t4;
                } else {
                    float v[P];
                    unpack_piece(t4, v);
                    store_piece(g, q, a.V, v);
                }
            }
        }
        if (W > 1) __syncthreads();
        if (W == 1) lds_phase();
    }
}

// Rows of any length, a workgroup of 8 waves each: one pass with a running maximum and sum per thread, and for the gradient
// a second one over the row (which the caches still hold in part).  Bound by reading the row: 2048 rows of 131071 bfloat16 classes, the loss
// alone, 112 us, 4.8 TB/s.
template <class T>
__global__ __launch_bounds__(512) void distill_stream_kernel(DistillArgs<T> a) {
    constexpr int P = kPiece<T>, THREADS = 512, WAVES = 8, AHEAD = 4;
    extern __shared__ unsigned member[];                  // a bit per class
    __shared__ float wave_max[WAVES];
    __shared__ double wave_part[WAVES];
    __shared__ float shared_coef;
    const int words = (a.V + 31) / 32, pieces = (a.V + P - 1) / P;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float c = kLog2e / a.t;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* p = a.x + row * a.ld;
        T* g = a.grad ? a.grad + row * a.ld_grad : nullptr;
        const float w = a.weight ? a.weight[row] : 1.0f;
        if (w == 0.0f) {
            if (tid == 0 && a.loss) a.loss[row] = 0.0f;
            float zeros[P] = {};
            if (g)
                for (int q = tid; q < pieces; q += THREADS) store_piece(g, q, a.V, zeros);
            continue;
        }
        int idx = -1;
        float z = 0.0f, s_k = -INFINITY;
        if (wave == 0 && lane < a.K) {
            idx = a.index[row * a.K + lane];
            z = a.values[row * a.K + lane];
        }
        for (int i = tid; i < words; i += THREADS) member[i] = 0;
        __syncthreads();
        const bool there = idx >= 0 && idx < a.V;
        bool again = false;
        if (there) {
            s_k = load_f32(p + idx);
            again = atomicOr(&member[idx >> 5], 1u << (idx & 31)) >> (idx & 31) & 1;
        }
        __syncthreads();
        float m_own = -INFINITY;
        double s_own = 0.0;
        for (int q = tid; q < pieces; q += THREADS * AHEAD) {
            uintx4 raw[AHEAD];
            float v[AHEAD][P];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) raw[i] = load_raw<false>(p, q + i * THREADS, a.V);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) unpack_piece(in_place<false>(raw[i], p, q + i * THREADS, a.V), v[i]);
            float m = m_own;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int at = (q + i * THREADS) * P;
                const unsigned bits = at < a.V ? member[at >> 5] >> (at & 31) : 0u;
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    v[i][e] = bits >> e & 1 ? -INFINITY : v[i][e];
                    m = fmaxf(m, v[i][e]);
                }
            }
            const float base = m == -INFINITY ? 0.0f : m;
            s_own = m_own == -INFINITY ? s_own : s_own * (double)__builtin_amdgcn_exp2f((m_own - base) * c);
            float part_own = 0.0f;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
#pragma unroll
                for (int e = 0; e < P; ++e) part_own += __builtin_amdgcn_exp2f((v[i][e] - base) * c);
            s_own += (double)part_own;
            m_own = m;
        }
        float m_r = group_max<64>(m_own);
        if (lane == 0) wave_max[wave] = m_r;
        __syncthreads();
        m_r = wave_max[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) m_r = fmaxf(m_r, wave_max[i]);
        const float base = m_r == -INFINITY ? 0.0f : m_r;
        const double part = group_sum<64>(m_own == -INFINITY ? s_own : s_own * (double)__builtin_amdgcn_exp2f((m_own - base) * c));
        if (lane == 0) wave_part[wave] = part;
        __syncthreads();
        if (wave == 0) {
            double sum_r = 0.0;
            for (int i = 0; i < WAVES; ++i) sum_r += wave_part[i];
            const double scale = (double)w * a.t;
            const double inv_t = 1.0 / a.t;
            const Teacher t = teacher_of<64>(there, z, a.lse != nullptr, a.lse ? a.lse[row] : 0.0f, inv_t);
            const RowResult r = row_result<64>(t, a.K, there, again, idx, s_k, a.lse != nullptr, inv_t, sum_r != sum_r ? NAN : m_r, sum_r, a.V);
            if (lane == 0) {
                if (a.loss) a.loss[row] = (float)(r.loss * scale * a.t);
                shared_coef = (float)(r.coef * scale);
            }
            if (g && r.first) store_f32(g + idx, (float)(r.grad_k * scale));
        }
        __syncthreads();
        if (g) {
            const float coef = shared_coef;
            for (int q = tid; q < pieces; q += THREADS) {
                float v[P];
                unpack_piece(in_place<false>(load_raw<false>(p, q, a.V), p, q, a.V), v);
#pragma unroll
                for (int e = 0; e < P; ++e) v[e] = coef != 0.0f ? coef * __builtin_amdgcn_exp2f((v[e] - base) * c) : 0.0f;
                const unsigned bits = member[q * P >> 5] >> (q * P & 31) & ((1u << P) - 1);
                if (bits == 0) {
                    store_piece(g, q, a.V, v);
                } else {                                  // the entries' own gradients are written above
#pragma unroll
                    for (int e = 0; e < P; ++e)
                        if (!(bits >> e & 1) && q * P + e < a.V) store_f32(g + q * P + e, v[e]);
                }
            }
        }
        __syncthreads();
    }
}

constexpr int64_t kMaxGrid = 1 << 20;          // workgroups of a launch; each walks the rows from there

// Rows of up to 128 classes: 16 lanes a row (97 float32 classes, 10 entries, 1.4M rows 328 us, a wave a row 793; 0.7M rows and
// 64 entries 455 against 703).
// Rows in LDS: one wave up to 6 KB (float32, 32 entries, 134M classes in all: 1100 classes 205 us against 287 of two waves,
// 1500 181 against 216, 2000 188 against 170), two up to 16 KB (4000 classes 135 against 162 of four, 203 of one), four up to
// 32 KB (6719 classes 120 against 165 of two).  More than 32 entries need a second wave's maxima for a useful bound, where
// the row has pieces for that many lanes (67M classes in all: 768 float32 classes, 64 entries 270 against 564); where it has
// hardly more pieces than entries, a lane's maxima are taken class by class (FEW: 500 bfloat16 classes, 64 entries 223 against
// 2212, 150 and 32 584 against 1069; with a few pieces more it costs: 500 and 32 180 against 123).  Beyond 32 KB, where a
// compute unit would hold few rows: eight waves on a row that is read twice (8000 float32 classes: 178 against 128 in LDS).
template <class T>
int launch_top(const TopArgs<T>& a, hipStream_t s) {
    const unsigned grid = (unsigned)std::min(a.rows, kMaxGrid);
    constexpr int P = kPiece<T>;
    const size_t row_lds = (size_t)(a.V + P - 1) / P * 16, found_lds = (size_t)a.K * 16 * sizeof(double);
    const unsigned groups = (unsigned)std::min<int64_t>((a.rows + 15) / 16, 2048);          // 8 per compute unit, which walk the rows
    if (a.V < P)                       // K <= V
        hipLaunchKernelGGL((top16_kernel<T, true>), dim3(groups), dim3(256), found_lds, s, a);
    else if (a.V <= kShort)
        hipLaunchKernelGGL((top16_kernel<T, false>), dim3(groups), dim3(256), found_lds, s, a);
    else if (row_lds < (size_t)(a.K > 32 ? 2 * a.K : a.K) * 16)          // less than 2 KB: K <= 64
        hipLaunchKernelGGL((top_lds_kernel<T, 1, 2, true>), dim3(grid), dim3(64), row_lds, s, a);
    else if (row_lds <= 6144 && (a.K <= 32 || row_lds < 2048)) {
        if (row_lds <= 2048)
            hipLaunchKernelGGL((top_lds_kernel<T, 1, 2>), dim3(grid), dim3(64), row_lds, s, a);
        else if (row_lds <= 4096)
            hipLaunchKernelGGL((top_lds_kernel<T, 1, 4>), dim3(grid), dim3(64), row_lds, s, a);
        else
            hipLaunchKernelGGL((top_lds_kernel<T, 1, 8>), dim3(grid), dim3(64), row_lds, s, a);
    } else if (row_lds <= kWaveBytes)
        hipLaunchKernelGGL((top_lds_kernel<T, 2, 8>), dim3(grid), dim3(128), row_lds, s, a);
    else if (row_lds <= kRowBytes)
        hipLaunchKernelGGL((top_lds_kernel<T, 4, 8>), dim3(grid), dim3(256), row_lds, s, a);
    else
        hipLaunchKernelGGL(top_stream_kernel<T>, dim3(grid), dim3(512), 0, s, a);
    OCR_HIP_CHECK(hipGetLastError());
    return OCRHIP_OK;
}

// Rows of up to 128 classes: 16, 32 or 64 lanes a row, as many as entries (97 float32 classes, 1.4M rows, 10 entries: 365 us
// against 1290 of a wave a row; 0.7M rows: 32 entries 298 against 666, 64 entries 568 against 681, where the row is also a
// wave's but the next one's loads are on their way).  Rows in LDS: one wave up to 16 KB (float32, 32 entries, 134M classes in
// all: 1000 classes 225 us against 404 of two waves, 2000 195 against 288; 4000 214 against 195; bfloat16 4000 classes 112
// against 157), four up to 32 KB (6719 classes 199 against 261 of one, 208 of two).  Beyond: eight waves on a row that is read
// twice (8000 float32 classes: 284 against 190 in LDS).
template <class T>
int launch_distill(const DistillArgs<T>& a, hipStream_t s) {
    constexpr int P = kPiece<T>;
    const size_t bits = (size_t)(a.V + 31) / 32 * 4, row_lds = (size_t)(a.V + P - 1) / P * 16;
    const unsigned grid = (unsigned)std::min(a.rows, kMaxGrid);
    const int lanes = a.K <= 16 ? 16 : a.K <= 32 ? 32 : 64;
    const unsigned groups = (unsigned)std::min<int64_t>((a.rows + 256 / lanes - 1) / (256 / lanes), 2048);   // 8 per compute unit, which walk the rows
    if (a.K <= 16 && a.V < P)
        hipLaunchKernelGGL((distill_short_kernel<T, true, 16>), dim3(groups), dim3(256), 0, s, a);
    else if (a.V >= P && a.V <= kShort) {
        if (lanes == 16)
            hipLaunchKernelGGL((distill_short_kernel<T, false, 16>), dim3(groups), dim3(256), 0, s, a);
        else if (lanes == 32)
            hipLaunchKernelGGL((distill_short_kernel<T, false, 32>), dim3(groups), dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL((distill_short_kernel<T, false, 64>), dim3(groups), dim3(256), 0, s, a);
    } else if (a.V < P)
        hipLaunchKernelGGL((distill_lds_kernel<T, 1, 1, true>), dim3(grid), dim3(64), row_lds, s, a);
    else if (row_lds <= 2048)
        hipLaunchKernelGGL((distill_lds_kernel<T, 1, 2, false>), dim3(grid), dim3(64), row_lds, s, a);
    else if (row_lds <= 4096)
        hipLaunchKernelGGL((distill_lds_kernel<T, 1, 4, false>), dim3(grid), dim3(64), row_lds, s, a);
    else if (row_lds <= kWaveBytes)
        hipLaunchKernelGGL((distill_lds_kernel<T, 1, 8, false>), dim3(grid), dim3(64), row_lds, s, a);
    else if (row_lds <= kRowBytes)
        hipLaunchKernelGGL((distill_lds_kernel<T, 4, 8, false>), dim3(grid), dim3(256), row_lds, s, a);
    else
        hipLaunchKernelGGL(distill_stream_kernel<T>, dim3(grid), dim3(512), bits, s, a);
    OCR_HIP_CHECK(hipGetLastError());
    return OCRHIP_OK;
}

}  // namespace

int launch_top_logits(const void* x, int dtype, int64_t rows, int V, int64_t ld, int K, float temperature, float* values, int* index, float* lse,
                      hipStream_t s) {
    if (rows == 0) return OCRHIP_OK;
    const double n = (double)rows * V;
    ProfScope prof("top_logits", 4.0 * n, n * (dtype == OCRHIP_F32 ? 4.0 : 2.0) + (double)rows * (8.0 * K + 4.0), s);
    const float inv_t = 1.0f / temperature;
    return dtype == OCRHIP_F32 ? launch_top(TopArgs<float>{(const float*)x, ld, rows, V, K, inv_t, values, index, lse}, s)
                               : launch_top(TopArgs<uint16_t>{(const uint16_t*)x, ld, rows, V, K, inv_t, values, index, lse}, s);
}

int launch_distill_loss(const void* x, int dtype, int64_t rows, int V, int64_t ld, const float* top_values, const int* top_index, int K, const float* top_lse,
                        float temperature, const float* weight, float* loss, void* grad, int64_t ld_grad, hipStream_t s) {
    if (rows == 0) return OCRHIP_OK;
    const double n = (double)rows * V, el = dtype == OCRHIP_F32 ? 4.0 : 2.0;
    ProfScope prof(grad ? "distill_loss<grad>" : "distill_loss", (grad ? 6.0 : 4.0) * n, n * el * (grad ? 2.0 : 1.0) + (double)rows * (8.0 * K + 4.0), s);
    if (dtype == OCRHIP_F32)
        return launch_distill(DistillArgs<float>{(const float*)x, ld, ld_grad, rows, top_values, top_lse, weight, top_index, loss, (float*)grad, V, K, temperature}, s);
    return launch_distill(DistillArgs<uint16_t>{(const uint16_t*)x, ld, ld_grad, rows, top_values, top_lse, weight, top_index, loss, (uint16_t*)grad, V, K, temperature}, s);
}

}  // namespace ocrhip
