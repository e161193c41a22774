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

template <class T>
__device__ __forceinline__ T wave_max(T v) {
    for (int o = 32; o; o >>= 1) {
        const T w = __shfl_xor(v, o);
        v = v > w ? v : w;
    }
    return v;
}
__device__ __forceinline__ float wave_fmax(float v) {
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// one workgroup per row, one pass over the row per entry
template <class T>
__global__ __launch_bounds__(256) void top_simple_kernel(const T* __restrict__ x, int64_t ld, int V, int K, float inv_t, float* __restrict__ values,
                                                         int* __restrict__ index, float* __restrict__ lse) {
    __shared__ unsigned long long best[4];
    __shared__ float fpart[4];
    const int64_t row = blockIdx.x;
    const T* p = x + row * ld;
    const int tid = threadIdx.x;
    unsigned long long last = ~0ull;
    float high = 0.0f;
    for (int k = 0; k < K; ++k) {
        unsigned long long mine = 0;
        for (int v = tid; v < V; v += 256) {
            const unsigned long long key = ((unsigned long long)order_key(load_f32(p + v)) << 32) | (0xFFFFFFFFu - (unsigned)v);
            if (key < last && key > mine) mine = key;
        }
        mine = wave_max(mine);
        __syncthreads();
        if ((tid & 63) == 0) best[tid >> 6] = mine;
        __syncthreads();
        last = max(max(best[0], best[1]), max(best[2], best[3]));
        const float value = key_value((unsigned)(last >> 32));
        if (k == 0) high = value;
        if (tid == 0) {
            values[row * K + k] = value;
            index[row * K + k] = (int)(0xFFFFFFFFu - (unsigned)last);
        }
    }
    if (!lse) return;
    float sum = 0.0f;
    for (int v = tid; v < V; v += 256) sum += expf((load_f32(p + v) - high) * inv_t);
    sum = wave_sum(sum);
    if ((tid & 63) == 0) fpart[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) lse[row] = fabsf(high) == INFINITY ? high : (float)((double)high * inv_t + log((double)fpart[0] + fpart[1] + fpart[2] + fpart[3]));
}

// What the K entries of a row and the sums over the rest (maximum m_r, sum of exp((s - m_r) / tau)) make of it.  One wave,
// lane k = entry k; float64 throughout.
struct RowResult {
    double loss;        // without weight and tau^2
    double coef;        // gradient of a class outside the entries = coef * exp((s - m_r) / tau)
    double grad_k;      // gradient of the lane's class (where the lane is its first entry)
    bool first;         // the lane's entry is there and no lower lane names its class
};
__device__ RowResult row_result(int lane, int K, bool there, int idx, float z, float s_k, bool has_lse, float t_lse, double inv_t, float m_r,
                                double sum_r, int V) {
    RowResult out;
    bool first = there;
    for (int j = 0; j < K; ++j) {
        const int other = __shfl(there ? idx : -1, j);
        if (j < lane && there && other == idx) first = false;
    }
    const float m_i = wave_fmax(first ? s_k : -INFINITY);
    const float m = fmaxf(m_r, m_i);
    const double d_k = ((double)s_k - m) * inv_t;
    const double e_k = first ? exp(d_k) : 0.0;
    const double shift = m_r == -INFINITY ? 0.0 : exp(((double)m_r - m) * inv_t);
    const double total = wave_sum(e_k) + sum_r * shift;
    const double log_total = log(total);
    const double log_q = d_k - log_total;
    const double zt = there ? (double)z * inv_t : -INFINITY;
    double log_p, p, rest = 0.0;
    bool teacher = true;
    if (has_lse) {
        log_p = zt - t_lse;
        p = exp(log_p);
        const double sum_p = wave_sum(p);
        rest = sum_p >= 1.0 ? 0.0 : 1.0 - sum_p;
        if (__popcll(__ballot(first)) == V) rest = 0.0;
    } else {
        const double top = wave_max(zt);
        teacher = top != -INFINITY || __ballot(zt != zt);
        const double e = exp(zt - top), sum_e = wave_sum(e);
        p = e / sum_e;
        log_p = zt - top - log(sum_e);
    }
    double loss = wave_sum(p == 0.0 ? 0.0 : p * (log_p - log_q));
    double coef = m_r == -INFINITY ? 0.0 : shift / total;
    if (has_lse && rest != 0.0) {
        const double log_rest = m_r == -INFINITY ? -INFINITY : log(sum_r) + ((double)m_r - m) * inv_t;
        loss += rest * (log(rest) - (log_rest - log_total));
        if (m_r != -INFINITY) coef -= rest / sum_r;
    }
    double sum_same = 0.0;
    for (int j = 0; j < K; ++j) {
        const int other = __shfl(there ? idx : -1, j);
        const double pj = __shfl(p, j);
        if (there && other == idx) sum_same += pj;
    }
    out.first = first;
    out.loss = teacher ? loss : 0.0;
    out.coef = !teacher ? 0.0 : loss != loss ? loss : coef;
    out.grad_k = !teacher ? 0.0 : loss != loss ? loss : exp(log_q) - sum_same;
    return out;
}

struct DistillArgs {
    const void* x;
    int64_t ld, ld_grad;
    const float *values, *lse, *weight;
    const int* index;
    float* loss;
    void* grad;
    int V, K;
    float t;
};

// one workgroup per row: maximum and sum over the classes outside the entries, the row's result, the gradient
template <class T>
__global__ __launch_bounds__(256) void distill_simple_kernel(DistillArgs a) {
    extern __shared__ unsigned member[];          // one bit per class
    __shared__ float fpart[4];
    __shared__ double shared_coef;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T* p = reinterpret_cast<const T*>(a.x) + row * a.ld;
    T* g = a.grad ? reinterpret_cast<T*>(a.grad) + row * a.ld_grad : nullptr;
    const float w = a.weight ? a.weight[row] : 1.0f;
    if (w == 0.0f) {
        if (tid == 0 && a.loss) a.loss[row] = 0.0f;
        if (g)
            for (int v = tid; v < a.V; v += 256) store_f32(g + v, 0.0f);
        return;
    }
    for (int i = tid; i < (a.V + 31) / 32; i += 256) member[i] = 0;
    __syncthreads();
    int idx = -1;
    float z = 0.0f, s_k = -INFINITY;
    if (wave == 0 && lane < a.K) {
        idx = a.index[row * a.K + lane];
        z = a.values[row * a.K + lane];
    }
    const bool there = idx >= 0 && idx < a.V;
    if (there) {
        s_k = load_f32(p + idx);
        atomicOr(&member[idx >> 5], 1u << (idx & 31));
    }
    __syncthreads();
    auto outside = [&](int v) { return !(member[v >> 5] >> (v & 31) & 1); };
    float m_r = -INFINITY;
    for (int v = tid; v < a.V; v += 256)
        if (outside(v)) m_r = fmaxf(m_r, load_f32(p + v));
    m_r = wave_fmax(m_r);
    if (lane == 0) fpart[wave] = m_r;
    __syncthreads();
    m_r = fmaxf(fmaxf(fpart[0], fpart[1]), fmaxf(fpart[2], fpart[3]));
    __syncthreads();
    const float base = m_r == -INFINITY ? 0.0f : m_r, inv_tf = 1.0f / a.t;
    float sum = 0.0f;
    for (int v = tid; v < a.V; v += 256)
        if (outside(v)) sum += expf((load_f32(p + v) - base) * inv_tf);
    sum = wave_sum(sum);
    if (lane == 0) fpart[wave] = sum;
    __syncthreads();
    const double sum_r = (double)fpart[0] + fpart[1] + fpart[2] + fpart[3];
    const double scale = (double)w * a.t;
    if (wave == 0) {
        // no finite class outside the entries, but a NaN among them: the maximum does not see it, the sum does
        const RowResult r = row_result(lane, a.K, there, idx, z, s_k, a.lse != nullptr, a.lse ? a.lse[row] : 0.0f, 1.0 / a.t, sum_r != sum_r ? NAN : m_r, sum_r, a.V);
        if (lane == 0) {
            if (a.loss) a.loss[row] = (float)(r.loss * scale * a.t);
            shared_coef = r.coef * scale;
        }
        if (g && r.first) store_f32(g + idx, (float)(r.grad_k * scale));
    }
    __syncthreads();
    if (!g) return;
    const float coef = (float)shared_coef;
    for (int v = tid; v < a.V; v += 256)
        if (outside(v)) store_f32(g + v, coef * expf((load_f32(p + v) - base) * inv_tf));
}

}  // namespace

int launch_top_logits(const void* x, int dtype, int64_t rows, int V, int64_t ld, int K, float temperature, float* values, int* index, float* lse,
                      hipStream_t s) {
    if (rows == 0) return OCRHIP_OK;
    const double n = (double)rows * V;
    ProfScope prof("top_logits", 4.0 * n, n * (dtype == OCRHIP_F32 ? 4.0 : 2.0) + (double)rows * (8.0 * K + 4.0), s);
    if (dtype == OCRHIP_F32)
        hipLaunchKernelGGL(top_simple_kernel<float>, dim3((unsigned)rows), dim3(256), 0, s, (const float*)x, ld, V, K, 1.0f / temperature, values, index, lse);
    else
        hipLaunchKernelGGL(top_simple_kernel<uint16_t>, dim3((unsigned)rows), dim3(256), 0, s, (const uint16_t*)x, ld, V, K, 1.0f / temperature, values, index, lse);
    OCR_HIP_CHECK(hipGetLastError());
    return OCRHIP_OK;
}

int launch_distill_loss(const void* x, int dtype, int64_t rows, int V, int64_t ld, const float* top_values, const int* top_index, int K, const float* top_lse,
                        float temperature, const float* weight, float* loss, void* grad, int64_t ld_grad, hipStream_t s) {
    if (rows == 0) return OCRHIP_OK;
    const double n = (double)rows * V, el = dtype == OCRHIP_F32 ? 4.0 : 2.0;
    ProfScope prof(grad ? "distill_loss<grad>" : "distill_loss", (grad ? 6.0 : 4.0) * n, n * el * (grad ? 2.0 : 1.0) + (double)rows * (8.0 * K + 4.0), s);
    DistillArgs a{x, ld, ld_grad, top_values, top_lse, weight, top_index, loss, grad, V, K, temperature};
    const size_t lds = (size_t)(V + 31) / 32 * 4;
    if (dtype == OCRHIP_F32)
        hipLaunchKernelGGL(distill_simple_kernel<float>, dim3((unsigned)rows), dim3(256), lds, s, a);
    else
        hipLaunchKernelGGL(distill_simple_kernel<uint16_t>, dim3((unsigned)rows), dim3(256), lds, s, a);
    OCR_HIP_CHECK(hipGetLastError());
    return OCRHIP_OK;
}

}  // namespace ocrhip
