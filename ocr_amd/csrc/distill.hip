// Distillation from a teacher's top logits (no counterpart in the reference, which holds no training code for this path):
// the K largest logits of a row with its log normaliser (the teacher's side), and the loss of a student's logits against
// them with its gradient.
//
//   entries k of a row: class i_k, logit z_k; temperature tau; student logits s
//   p_k = softmax of z / tau over the entries, or, with the teacher's lse = log sum_v exp(z_v / tau),
//   p_k = exp(z_k / tau - lse) and one more class p_rest = 1 - sum p_k for everything outside the entries
//   q   = softmax(s / tau);  q_rest = sum of q outside the entries
//   loss = w tau^2 (sum_k p_k log(p_k / q_(i_k)) [+ p_rest log(p_rest / q_rest)])
//   d loss / d s_v = w tau (q_v - p_v) for the entries, w tau q_v (1 [- p_rest / q_rest]) outside them
//
// Where teacher and student nearly agree the loss is far smaller than the terms it is the sum of.  The sums over the
// classes outside the entries are float32: an error there changes the loss only in proportion to q_rest - p_rest.  What
// enters to first order (the entries' probabilities, the logarithms, the sum of the terms: K numbers per row) is float64.
#include <algorithm>

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

// ---- reductions over groups of 16 or 64 lanes, on the vector ALU: quad, half row and row exchanges, then the swaps of
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
    if (G == 64) {
        T a, b;
        swapped<false>(v, a, b);
        v = op(a, b);
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
__device__ __forceinline__ double group_max(double v) { return reduce<G>(v, [](double a, double b) { return fmax(a, b); }); }
template <int G>
__device__ __forceinline__ unsigned group_max(unsigned v) { return reduce<G>(v, [](unsigned a, unsigned b) { return a > b ? a : b; }); }
template <int G>
__device__ __forceinline__ unsigned group_min(unsigned v) { return reduce<G>(v, [](unsigned a, unsigned b) { return a < b ? a : b; }); }
// the ballot of the lane's group
template <int G>
__device__ __forceinline__ unsigned long long group_ballot(bool b) {
    const unsigned long long w = __ballot(b);
    return G == 64 ? w : w >> (threadIdx.x & 48) & 0xFFFFull;
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

// piece c of a row of V; classes from V on are -infinity
__device__ __forceinline__ void load_piece(const float* p, int c, int V, float* v) {
    if (c * 4 + 4 <= V) {
        const floatx4 t = *reinterpret_cast<const floatx4_any*>(p + c * 4);
        v[0] = t[0]; v[1] = t[1]; v[2] = t[2]; v[3] = t[3];
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = c * 4 + e < V ? p[c * 4 + e] : -INFINITY;
}
__device__ __forceinline__ void load_piece(const uint16_t* p, int c, int V, float* v) {
    if (c * 8 + 8 <= V) {
        const uintx4 t = *reinterpret_cast<const uintx4_any*>(p + c * 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(t[i] << 16);
            v[2 * i + 1] = __uint_as_float(t[i] & 0xFFFF0000u);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c * 8 + e < V ? load_f32(p + c * 8 + e) : -INFINITY;
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

// ---- top logits
//
// Bound by reading the logits once.  Rows of up to 128 classes and 16 entries: 16 lanes per row, the maximum taken away K
// times.  Longer rows: the K-th largest of the lanes' own maxima is a lower bound of the K-th largest of all (K lanes hold
// a value that large), and hardly more than K values reach it: it is found by bisection of its leading bits, the values
// that reach it are put on a list in LDS and each finds its rank by counting the larger ones.  A row whose list overflows
// (thousands of equal values) takes its maxima one by one.
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

__device__ __forceinline__ float row_lse(float high, float inv_t, double sum) {
    return fabsf(high) == INFINITY ? high : (float)((double)high * inv_t + log(sum));
}

template <class T>
__global__ __launch_bounds__(256) void top16_kernel(TopArgs<T> a) {
    constexpr int P = kPiece<T>, N = 128 / 16 / P;
    const int part = threadIdx.x & 15;
    for (int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); row < a.rows; row += (int64_t)gridDim.x * 16) {
        const T* p = a.x + row * a.ld;
        float v[N][P];
        unsigned key[N][P];
        unsigned best = 0, at = 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < N; ++i) load_piece(p, part + 16 * i, a.V, v[i]);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < P; ++e) key[i][e] = (part + 16 * i) * P + e < a.V ? order_key(v[i][e]) : 0u;
        float high = 0.0f;
        for (int k = 0; k < a.K; ++k) {
            best = 0;
            at = 0xFFFFFFFFu;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e < P; ++e)
                    if (key[i][e] > best) {
                        best = key[i][e];
                        at = (part + 16 * i) * P + e;
                    }
            const unsigned top = group_max<16>(best);
            const unsigned where = group_min<16>(best == top ? at : 0xFFFFFFFFu);
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e < P; ++e)
                    if ((unsigned)((part + 16 * i) * P + e) == where) key[i][e] = 0;
            if (k == 0) high = key_value(top);
            if (part == 0) {
                a.values[row * a.K + k] = key_value(top);
                a.index[row * a.K + k] = (int)where;
            }
        }
        if (a.lse) {
            const float c = a.inv_t * kLog2e;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e < P; ++e) sum += __builtin_amdgcn_exp2f((v[i][e] - high) * c);
            sum = group_sum<16>(sum);
            if (part == 0) a.lse[row] = row_lse(high, a.inv_t, (double)sum);
        }
    }
}

constexpr int kTopList = 512;          // candidates of a row that LDS holds

// WAVES waves per row.  HELD > 0: pieces per thread kept in registers (rows of up to 64 * WAVES * HELD pieces, one read);
// 0: the row is read twice, for the lanes' maxima and for the values that reach the bound.
template <class T, int WAVES, int HELD>
__global__ __launch_bounds__(WAVES * 64) void top_kernel(TopArgs<T> a) {
    constexpr int P = kPiece<T>, THREADS = WAVES * 64, KEEP = HELD ? HELD : 1, AHEAD = 4;
    __shared__ unsigned long long list[kTopList];
    __shared__ unsigned maxima[THREADS];
    __shared__ float wave_sum[WAVES];
    __shared__ unsigned long long wave_best[WAVES];
    __shared__ unsigned shared_bound;
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int pieces = (a.V + P - 1) / P;
    const float c = a.inv_t * kLog2e;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* p = a.x + row * a.ld;
        float v[KEEP][P];
        unsigned mine = 0;
        float m_own = -INFINITY, s_own = 0.0f;          // HELD 0: running maximum and sum of the thread
        if (tid == 0) count = 0;
        if constexpr (HELD > 0) {
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                if (tid + i * THREADS < pieces)
                    load_piece(p, tid + i * THREADS, a.V, v[i]);
                else
#pragma unroll
                    for (int e = 0; e < P; ++e) v[i][e] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < HELD; ++i)
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    const unsigned k = (tid + i * THREADS) * P + e < a.V ? order_key(v[i][e]) : 0u;
                    mine = max(mine, k);
                }
        } else {
            for (int q = tid; q < pieces; q += THREADS * AHEAD) {
                float w[AHEAD][P];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    if (q + i * THREADS < pieces)
                        load_piece(p, q + i * THREADS, a.V, w[i]);
                    else
#pragma unroll
                        for (int e = 0; e < P; ++e) w[i][e] = -INFINITY;
                }
                float m = m_own;
#pragma unroll
                for (int i = 0; i < AHEAD; ++i)
#pragma unroll
                    for (int e = 0; e < P; ++e) {
                        const unsigned k = (q + i * THREADS) * P + e < a.V ? order_key(w[i][e]) : 0u;
                        mine = max(mine, k);
                        m = fmaxf(m, w[i][e]);
                    }
                const float base = m == -INFINITY ? 0.0f : m;
                s_own = m_own == -INFINITY ? 0.0f : s_own * __builtin_amdgcn_exp2f((m_own - base) * c);
#pragma unroll
                for (int i = 0; i < AHEAD; ++i)
#pragma unroll
                    for (int e = 0; e < P; ++e) s_own += __builtin_amdgcn_exp2f((w[i][e] - base) * c);
                m_own = m;
            }
        }
        maxima[tid] = mine;
        __syncthreads();
        if (wave == 0) {
            // the largest bound of 20 leading bits that K of the maxima reach
            unsigned m[WAVES], top = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                m[w] = maxima[w * 64 + lane];
                top = max(top, m[w]);
            }
            unsigned bound = 0;
            for (int bit = 31; bit >= 12; --bit) {
                const unsigned next = bound | 1u << bit;
                int reach = 0;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) reach += __popcll(__ballot(m[w] >= next));
                if (reach >= a.K) bound = next;
            }
            top = group_max<64>(top);
            if (lane == 0) {
                shared_bound = max(bound, 1u);
                wave_best[0] = top;
            }
        }
        __syncthreads();
        const unsigned bound = shared_bound;
        const float high = key_value((unsigned)wave_best[0]);
        // the values that reach the bound
        auto offer = [&](float x, int at) {
            const unsigned k = order_key(x);
            if (k >= bound && at < a.V) {
                const int slot = atomicAdd(&count, 1);
                if (slot < kTopList) list[slot] = (unsigned long long)k << 32 | (0xFFFFFFFFu - (unsigned)at);
            }
        };
        if (mine >= bound) {
            if constexpr (HELD > 0) {
#pragma unroll
                for (int i = 0; i < HELD; ++i)
#pragma unroll
                    for (int e = 0; e < P; ++e) offer(v[i][e], (tid + i * THREADS) * P + e);
            } else {
                for (int q = tid; q < pieces; q += THREADS) {
                    float w[P];
                    load_piece(p, q, a.V, w);
#pragma unroll
                    for (int e = 0; e < P; ++e) offer(w[e], q * P + e);
                }
            }
        }
        if (a.lse) {
            float sum = 0.0f;
            if constexpr (HELD > 0) {
#pragma unroll
                for (int i = 0; i < HELD; ++i)
#pragma unroll
                    for (int e = 0; e < P; ++e) sum += __builtin_amdgcn_exp2f((v[i][e] - high) * c);
            } else {
                sum = m_own == -INFINITY ? s_own : s_own * __builtin_amdgcn_exp2f((m_own - high) * c);
            }
            sum = group_sum<64>(sum);
            if (lane == 0) wave_sum[wave] = sum;
        }
        __syncthreads();
        const int n = count;
        if (n <= kTopList) {
            for (int i = tid; i < n; i += THREADS) {
                const unsigned long long own = list[i];
                int rank = 0;
                for (int j = 0; j < n; ++j) rank += list[j] > own ? 1 : 0;
                if (rank < a.K) {
                    a.values[row * a.K + rank] = key_value((unsigned)(own >> 32));
                    a.index[row * a.K + rank] = (int)(0xFFFFFFFFu - (unsigned)own);
                }
            }
        } else {
            unsigned long long last = ~0ull;
            for (int k = 0; k < a.K; ++k) {
                unsigned long long best = 0;
                for (int at = tid; at < a.V; at += THREADS) {
                    const unsigned long long key = (unsigned long long)order_key(load_f32(p + at)) << 32 | (0xFFFFFFFFu - (unsigned)at);
                    if (key < last && key > best) best = key;
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
        if (a.lse && tid == 0) {
            double sum = 0.0;
            for (int w = 0; w < WAVES; ++w) sum += (double)wave_sum[w];
            a.lse[row] = row_lse(high, a.inv_t, sum);
        }
        __syncthreads();
    }
}

// ---- distillation

// What the K entries of a row and the sums over the rest (maximum m_r, sum of exp((s - m_r) / tau)) make of it.  A group of
// G lanes (16 or 64, K <= G), lane k = entry k; float64 throughout.
struct RowResult {
    double loss;        // without weight and tau^2
    double coef;        // gradient of a class outside the entries = coef * exp((s - m_r) / tau)
    double grad_k;      // gradient of the lane's class (where the lane is its first entry)
    bool first;         // the lane's entry is there and no lower lane names its class
};
template <int G>
__device__ RowResult row_result(int K, bool there, bool again, int idx, float z, float s_k, bool has_lse, float t_lse, double inv_t, float m_r,
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
    const float m_i = group_max<G>(first ? s_k : -INFINITY);
    const float m = fmaxf(m_r, m_i);
    const double d_k = ((double)s_k - m) * inv_t;
    const double e_k = first ? exp(d_k) : 0.0;
    const double shift = m_r == -INFINITY ? 0.0 : exp(((double)m_r - m) * inv_t);
    const double total = group_sum<G>(e_k) + sum_r * shift;
    const double log_total = log(total);
    const double log_q = d_k - log_total;
    const double zt = there ? (double)z * inv_t : -INFINITY;
    double log_p, p, rest = 0.0;
    bool teacher = true;
    if (has_lse) {
        log_p = zt - t_lse;
        p = exp(log_p);
        const double sum_p = group_sum<G>(p);
        rest = sum_p >= 1.0 ? 0.0 : 1.0 - sum_p;
        if (__popcll(group_ballot<G>(first)) == V) rest = 0.0;
    } else {
        const double top = group_max<G>(zt);
        teacher = top != -INFINITY || group_ballot<G>(zt != zt) != 0;
        const double e = exp(zt - top), sum_e = group_sum<G>(e);
        p = e / sum_e;
        log_p = zt - top - log(sum_e);
    }
    double loss = group_sum<G>(p == 0.0 ? 0.0 : p * (log_p - log_q));
    double coef = m_r == -INFINITY ? 0.0 : shift / total;
    if (has_lse && rest != 0.0) {
        const double log_rest = m_r == -INFINITY ? -INFINITY : log(sum_r) + ((double)m_r - m) * inv_t;
        loss += rest * (log(rest) - (log_rest - log_total));
        if (m_r != -INFINITY) coef -= rest / sum_r;
    }
    double sum_same = p;
    if (doubled) {
        sum_same = 0.0;
        for (int j = 0; j < K; ++j) {
            const int other = __shfl(there ? idx : -1, j, G);
            const double pj = __shfl(p, j, G);
            if (there && other == idx) sum_same += pj;
        }
    }
    out.first = first;
    out.loss = teacher ? loss : 0.0;
    out.coef = !teacher ? 0.0 : loss != loss ? loss : coef;
    out.grad_k = !teacher ? 0.0 : loss != loss ? loss : exp(log_q) - sum_same;
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

// A row in registers: pieces lane + i * LANES, i < N, of LANES lanes (or threads) share it.
template <class T, int LANES, int N>
struct RowPieces {
    static constexpr int P = kPiece<T>;
    float v[N][P];
    __device__ __forceinline__ void load(const T* p, int part, int V) {
        const int pieces = (V + P - 1) / P;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (part + i * LANES < pieces)
                load_piece(p, part + i * LANES, V, v[i]);
            else
#pragma unroll
                for (int e = 0; e < P; ++e) v[i][e] = -INFINITY;
        }
    }
    // the classes that are entries (a bit each) leave the sums; returns the lane's maximum of the rest
    __device__ __forceinline__ float mask(const unsigned* member, int part, int V) {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (part + i * LANES) * P;
            const unsigned bits = at < V ? member[at >> 5] >> (at & 31) : 0u;
#pragma unroll
            for (int e = 0; e < P; ++e) {
                v[i][e] = bits >> e & 1 ? -INFINITY : v[i][e];
                m = fmaxf(m, v[i][e]);
            }
        }
        return m;
    }
    // v = exp((v - base) / tau), c = log2 e / tau; returns the lane's sum
    __device__ __forceinline__ float exponentials(float base, float c) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int e = 0; e < P; ++e) {
                v[i][e] = __builtin_amdgcn_exp2f((v[i][e] - base) * c);
                sum += v[i][e];
            }
        }
        return sum;
    }
    // gradient: coef * v outside the entries (0 for coef 0, whatever v is), the value of `inside` (by class) for them
    __device__ __forceinline__ void store(T* g, int part, int V, const unsigned* member, const float* inside, float coef) {
        const int pieces = (V + P - 1) / P;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (part + i * LANES >= pieces) break;
            const int at = (part + i * LANES) * P;
            const unsigned bits = member[at >> 5] >> (at & 31) & ((1u << P) - 1);
            float o[P];
#pragma unroll
            for (int e = 0; e < P; ++e) o[e] = coef != 0.0f ? coef * v[i][e] : 0.0f;
            if (bits)
#pragma unroll
                for (int e = 0; e < P; ++e)
                    if (bits >> e & 1) o[e] = inside[at + e];
            store_piece(g, part + i * LANES, V, o);
        }
    }
    __device__ __forceinline__ void store_zeros(T* g, int part, int V) {
        const int pieces = (V + P - 1) / P;
        float o[P];
#pragma unroll
        for (int e = 0; e < P; ++e) o[e] = 0.0f;
        for (int q = part; q < pieces; q += LANES) store_piece(g, q, V, o);
    }
};

// G lanes of one wave per row (rows of up to CAP classes): the row is read once and stays in registers, its entries' bits
// and gradients are in LDS of the group's own, nothing waits for another wave.
template <class T, int G, int CAP>
__global__ __launch_bounds__(256) void distill_group_kernel(DistillArgs<T> a) {
    constexpr int ROWS = 256 / G, WORDS = CAP / 32;
    __shared__ unsigned member_all[ROWS][WORDS];
    __shared__ float inside_all[ROWS][CAP];
    const int part = threadIdx.x & (G - 1), sub = threadIdx.x / G;
    unsigned* member = member_all[sub];
    float* inside = inside_all[sub];
    const double inv_t = 1.0 / a.t;
    const float c = kLog2e / a.t;
    RowPieces<T, G, CAP / G / kPiece<T>> row_v;
    for (int64_t first_row = (int64_t)blockIdx.x * ROWS; first_row < a.rows; first_row += (int64_t)gridDim.x * ROWS) {
        const int64_t row = first_row + sub;
        const bool in_range = row < a.rows;
        const float w = !in_range ? 0.0f : a.weight ? a.weight[row] : 1.0f;
        const T* p = a.x + row * a.ld;
        const bool live = w != 0.0f;               // the others of the wave may be: everything below runs for all lanes
        if (live) row_v.load(p, part, a.V);
        int idx = -1;
        float z = 0.0f, s_k = -INFINITY;
        if (live && part < a.K) {
            idx = a.index[row * a.K + part];
            z = a.values[row * a.K + part];
        }
        const bool there = idx >= 0 && idx < a.V;
        for (int i = part; i < WORDS; i += G) member[i] = 0;
        __builtin_amdgcn_wave_barrier();
        bool again = false;
        if (there) {
            s_k = load_f32(p + idx);
            again = atomicOr(&member[idx >> 5], 1u << (idx & 31)) >> (idx & 31) & 1;
        }
        __builtin_amdgcn_wave_barrier();
        const float m_r = group_max<G>(row_v.mask(member, part, a.V));
        const float base = m_r == -INFINITY ? 0.0f : m_r;
        const float sum_r = group_sum<G>(row_v.exponentials(base, c));
        // no finite class outside the entries, but a NaN among them: the maximum does not see it, the sum does
        const RowResult r = row_result<G>(a.K, there, again, idx, z, s_k, a.lse != nullptr, a.lse && live ? a.lse[row] : 0.0f, inv_t, sum_r != sum_r ? NAN : m_r,
                                          (double)sum_r, a.V);
        const double scale = (double)w * a.t;
        if (a.loss && in_range && part == 0) a.loss[row] = live ? (float)(r.loss * scale * a.t) : 0.0f;
        if (a.grad && in_range) {
            T* g = a.grad + row * a.ld_grad;
            if (live) {
                if (r.first) inside[idx] = (float)(r.grad_k * scale);
                __builtin_amdgcn_wave_barrier();
                row_v.store(g, part, a.V, member, inside, (float)(r.coef * scale));
            } else {
                row_v.store_zeros(g, part, a.V);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// A workgroup of 4 waves per row of up to 8192 classes, the row in registers.
constexpr int kBlockClasses = 8192;
template <class T>
__global__ __launch_bounds__(256) void distill_block_kernel(DistillArgs<T> a) {
    extern __shared__ unsigned dynamic_lds[];             // a bit per class, then (for the gradient) a float per class
    __shared__ float wave_part[4];
    __shared__ float shared_coef;
    const int words = (a.V + 31) / 32;
    unsigned* member = dynamic_lds;
    float* inside = reinterpret_cast<float*>(dynamic_lds + words);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float c = kLog2e / a.t;
    RowPieces<T, 256, kBlockClasses / 256 / kPiece<T>> row_v;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* p = a.x + row * a.ld;
        T* g = a.grad ? a.grad + row * a.ld_grad : nullptr;
        const float w = a.weight ? a.weight[row] : 1.0f;
        if (w == 0.0f) {
            if (tid == 0 && a.loss) a.loss[row] = 0.0f;
            if (g) row_v.store_zeros(g, tid, a.V);
            continue;
        }
        row_v.load(p, tid, a.V);
        int idx = -1;
        float z = 0.0f, s_k = -INFINITY;
        if (wave == 0 && lane < a.K) {
            idx = a.index[row * a.K + lane];
            z = a.values[row * a.K + lane];
        }
        for (int i = tid; i < words; i += 256) member[i] = 0;
        __syncthreads();
        const bool there = idx >= 0 && idx < a.V;
        bool again = false;
        if (there) {
            s_k = load_f32(p + idx);
            again = atomicOr(&member[idx >> 5], 1u << (idx & 31)) >> (idx & 31) & 1;
        }
        __syncthreads();
        float m_r = group_max<64>(row_v.mask(member, tid, a.V));
        if (lane == 0) wave_part[wave] = m_r;
        __syncthreads();
        m_r = fmaxf(fmaxf(wave_part[0], wave_part[1]), fmaxf(wave_part[2], wave_part[3]));
        const float base = m_r == -INFINITY ? 0.0f : m_r;
        const float part = group_sum<64>(row_v.exponentials(base, c));
        __syncthreads();
        if (lane == 0) wave_part[wave] = part;
        __syncthreads();
        if (wave == 0) {
            const double sum_r = (double)wave_part[0] + wave_part[1] + wave_part[2] + wave_part[3], scale = (double)w * a.t;
            const RowResult r = row_result<64>(a.K, there, again, idx, z, s_k, a.lse != nullptr, a.lse ? a.lse[row] : 0.0f, 1.0 / a.t, sum_r != sum_r ? NAN : m_r, sum_r, a.V);
            if (lane == 0) {
                if (a.loss) a.loss[row] = (float)(r.loss * scale * a.t);
                shared_coef = (float)(r.coef * scale);
            }
            if (g && r.first) inside[idx] = (float)(r.grad_k * scale);
        }
        if (!g) {
            __syncthreads();
            continue;
        }
        __syncthreads();
        row_v.store(g, tid, a.V, member, inside, shared_coef);
        __syncthreads();
    }
}

// Rows of any length, a workgroup of 8 waves each: one pass with a running maximum and sum per thread, and for the gradient
// a second one over the row (which the caches still hold in part).
template <class T>
__global__ __launch_bounds__(512) void distill_stream_kernel(DistillArgs<T> a) {
    constexpr int P = kPiece<T>, THREADS = 512, WAVES = 8, AHEAD = 4;
    extern __shared__ unsigned member[];                  // a bit per class
    __shared__ float wave_max[WAVES], wave_part[WAVES];
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
        float m_own = -INFINITY, s_own = 0.0f;
        for (int q = tid; q < pieces; q += THREADS * AHEAD) {
            float v[AHEAD][P];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                if (q + i * THREADS < pieces)
                    load_piece(p, q + i * THREADS, a.V, v[i]);
                else
#pragma unroll
                    for (int e = 0; e < P; ++e) v[i][e] = -INFINITY;
            }
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
            s_own = m_own == -INFINITY ? s_own : s_own * __builtin_amdgcn_exp2f((m_own - base) * c);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
#pragma unroll
                for (int e = 0; e < P; ++e) s_own += __builtin_amdgcn_exp2f((v[i][e] - base) * c);
            m_own = m;
        }
        float m_r = group_max<64>(m_own);
        if (lane == 0) wave_max[wave] = m_r;
        __syncthreads();
        m_r = wave_max[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) m_r = fmaxf(m_r, wave_max[i]);
        const float base = m_r == -INFINITY ? 0.0f : m_r;
        const float part = group_sum<64>(m_own == -INFINITY ? s_own : s_own * __builtin_amdgcn_exp2f((m_own - base) * c));
        if (lane == 0) wave_part[wave] = part;
        __syncthreads();
        if (wave == 0) {
            double sum_r = 0.0;
            for (int i = 0; i < WAVES; ++i) sum_r += (double)wave_part[i];
            const double scale = (double)w * a.t;
            const RowResult r = row_result<64>(a.K, there, again, idx, z, s_k, a.lse != nullptr, a.lse ? a.lse[row] : 0.0f, 1.0 / a.t, sum_r != sum_r ? NAN : m_r, sum_r, a.V);
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
                load_piece(p, q, a.V, v);
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

template <class T>
int launch_top(const TopArgs<T>& a, hipStream_t s) {
    const unsigned grid = (unsigned)std::min(a.rows, kMaxGrid);
    constexpr int P = kPiece<T>;
    if (a.V <= 128 && a.K <= 16)
        hipLaunchKernelGGL(top16_kernel<T>, dim3((unsigned)std::min((a.rows + 15) / 16, kMaxGrid)), dim3(256), 0, s, a);
    else if (a.V <= 1024)
        hipLaunchKernelGGL((top_kernel<T, 1, 1024 / 64 / P>), dim3(grid), dim3(64), 0, s, a);
    else if (a.V <= kBlockClasses)
        hipLaunchKernelGGL((top_kernel<T, 4, kBlockClasses / 256 / P>), dim3(grid), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((top_kernel<T, 8, 0>), dim3(grid), dim3(512), 0, s, a);
    OCR_HIP_CHECK(hipGetLastError());
    return OCRHIP_OK;
}

template <class T>
int launch_distill(const DistillArgs<T>& a, hipStream_t s) {
    const size_t bits = (size_t)(a.V + 31) / 32 * 4;
    const unsigned grid = (unsigned)std::min(a.rows, kMaxGrid);
    if (a.V <= 128 && a.K <= 16)
        hipLaunchKernelGGL((distill_group_kernel<T, 16, 128>), dim3((unsigned)std::min((a.rows + 15) / 16, kMaxGrid)), dim3(256), 0, s, a);
    else if (a.V <= 1024)
        hipLaunchKernelGGL((distill_group_kernel<T, 64, 1024>), dim3((unsigned)std::min((a.rows + 3) / 4, kMaxGrid)), dim3(256), 0, s, a);
    else if (a.V <= kBlockClasses)
        hipLaunchKernelGGL(distill_block_kernel<T>, dim3(grid), dim3(256), bits + (a.grad ? (size_t)a.V * 4 : 0), s, a);
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
