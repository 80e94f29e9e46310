// Distillation from a teacher's largest logits: their selection, and the loss of a student against them with its gradient.
//
// Logits lie as [outer][classes][inner] (inner = 1: rows of logits, which may be `ld` elements apart; inner > 1: maps
// [N, C, H * W]); a "row" is one (outer, inner) position.
//
// Selection: the k largest logits of a row in descending order, equal ones by ascending index, NaN above every number; and
//   rest = log sum over the OTHERS of exp(logit / T)          (-inf when nothing is left)
// so that values and rest together hold the teacher's whole distribution up to the split of the rest.
//
// Loss of a row with teacher entries (v_i, idx_i) and rest; z the student's logits, a_j = z_j / T:
//   p_i = exp(v_i / T - L), p_r = exp(rest - L), L = log(sum_i exp(v_i / T) + exp(rest));   q = softmax(a),
//   q_r = q's mass outside the listed classes
//   loss = T^2 [ sum_i p_i (log p_i - log q_idx_i) + p_r (log p_r - log q_r) ],   0 log 0 = 0
//   d loss / d z_j = T (q_j - sum_{i: idx_i = j} p_i)                              listed classes
//                  = T r_j (q_r - p_r),  r_j = the share of class j in q_r        all others
// The others' form is T (q_j - p_r r_j) with the common factor taken out: one exponential per element, and no cancellation
// between q_j and p_r r_j beyond that of the two row constants.  q_r is summed over the unlisted classes themselves (1 minus
// the listed ones would lose it where the student is sure).
// Entries with a negative index are padding.  A row counts when its mask is set (or there is none) and its teacher holds
// anything (L > -inf); other rows have no loss and a zero gradient, whatever they hold.  A softmax over nothing is zero
// everywhere.  An index past the classes makes the row's loss and gradient NaN and reads nothing.
#include "common.h"
#include "../../include/msfwsi_hip.h"

namespace {

constexpr int kT = 256;
constexpr int kMaxK = 64;

// fp32 -> int of the same order; -0 equals +0, every NaN is the largest
__device__ __forceinline__ int order_of(float x) {
    if (x != x) return 0x7fffffff;
    const int b = (int)__float_as_uint(x + 0.f);
    return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float value_of(int order) {  // 0x80000000, below every number, stands for nothing: -inf
    if (order == (int)0x80000000) return -INFINITY;
    return __uint_as_float((unsigned)(order ^ ((order >> 31) & 0x7fffffff)));
}
__device__ __forceinline__ long key_of(float x, int idx) { return ((long)order_of(x) << 32) | (unsigned)(0x7fffffff - idx); }

template <typename V, typename OP>
__device__ __forceinline__ V block_all(V v, V* buf, OP op) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = op(v, __shfl_xor(v, off, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
    __syncthreads();
    v = buf[0];
    for (int i = 1; i < kT / 64; ++i) v = op(v, buf[i]);
    return v;
}
struct OpMax {
    __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
    __device__ long operator()(long a, long b) const { return a > b ? a : b; }
};
struct OpAdd {
    __device__ float operator()(float a, float b) const { return a + b; }
};

template <typename T>
__global__ void __launch_bounds__(kT) top_logits_kernel(const T* __restrict__ x, long ld, int C, long inner, int k, float inv_t,
                                                        float* __restrict__ values, int* __restrict__ indices, float* __restrict__ rest) {
    __shared__ long lbuf[kT / 64];
    __shared__ float fbuf[kT / 64];
    const long o = blockIdx.x / inner, i = blockIdx.x % inner;
    const T* p = x + o * ld + i;
    long last = 0x7fffffffffffffffL;
    for (int s = 0; s < k; ++s) {
        long best = (long)0x8000000000000000L;
        for (int c = threadIdx.x; c < C; c += kT) {
            const long key = key_of(load_elem<T>(p, c * inner), c);
            if (key < last && key > best) best = key;
        }
        last = block_all(best, lbuf, OpMax());
        if (threadIdx.x == 0) {
            const int c = 0x7fffffff - (int)(unsigned)last;
            values[(o * k + s) * inner + i] = load_elem<T>(p, c * inner);
            indices[(o * k + s) * inner + i] = c;
        }
    }
    long most = (long)0x8000000000000000L;  // the largest of the others, NaN on top
    float sum = 0.f;
    for (int c = threadIdx.x; c < C; c += kT) {
        const long key = key_of(load_elem<T>(p, c * inner), c);
        if (key < last && key > most) most = key;
    }
    most = block_all(most, lbuf, OpMax());
    const float top = value_of((int)(most >> 32));
    const float m = top == -INFINITY ? 0.f : top;
    for (int c = threadIdx.x; c < C; c += kT) {
        const float v = load_elem<T>(p, c * inner);
        if (key_of(v, c) < last) sum += expf((v - m) * inv_t);
    }
    sum = block_all(sum, fbuf, OpAdd());
    if (threadIdx.x == 0) rest[blockIdx.x] = top == INFINITY ? top : m * inv_t + logf(sum);
}

// the teacher's distribution of one row, in LDS: p[i] (0 for padding), p_r; false when the row holds nothing
struct Teacher {
    float p[kMaxK], logp[kMaxK];
    int idx[kMaxK];
    float pr, logpr;
    int holds, bad;
};
__device__ __forceinline__ void teacher_row(Teacher& t, const float* __restrict__ values, const int* __restrict__ indices,
                                            const float* __restrict__ rest, long row, long o, long i, long inner, int k, int C, float inv_t) {
    if (threadIdx.x == 0) {
        float top = -INFINITY, sum = 0.f;
        int bad = 0;
        const float r = rest != nullptr ? rest[row] : -INFINITY;
        top = r;
        for (int s = 0; s < k; ++s) {
            const int c = indices[(o * k + s) * inner + i];
            const float v = c < 0 ? -INFINITY : values[(o * k + s) * inner + i] * inv_t;
            bad |= c >= C;
            t.idx[s] = c;
            t.logp[s] = v;
            top = v != v ? v : v > top ? v : top;
        }
        const float m = top == -INFINITY ? 0.f : top;
        for (int s = 0; s < k; ++s) sum += expf(t.logp[s] - m);
        sum += expf(r - m);
        const float L = m + logf(sum);
        for (int s = 0; s < k; ++s) {
            t.logp[s] -= L;
            t.p[s] = expf(t.logp[s]);
        }
        t.logpr = r - L;
        t.pr = expf(t.logpr);
        t.holds = top != -INFINITY;
        t.bad = bad;
    }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kT) distill_fwd_kernel(const T* __restrict__ z, long ld, int C, long inner, int k,
                                                         const float* __restrict__ values, const int* __restrict__ indices,
                                                         const float* __restrict__ rest, const unsigned char* __restrict__ mask, float temp,
                                                         float inv_t, float4* __restrict__ stats, float* __restrict__ row_loss) {
    __shared__ Teacher t;
    __shared__ float buf[kT / 64];
    const long row = blockIdx.x, o = row / inner, i = row % inner;
    teacher_row(t, values, indices, rest, row, o, i, inner, k, C, inv_t);
    if (!t.holds || (mask != nullptr && mask[row] == 0)) {
        if (threadIdx.x == 0) stats[row] = make_float4(0.f, 0.f, 0.f, 0.f), row_loss[row] = 0.f;
        return;
    }
    const T* p = z + o * ld + i;
    float top = -INFINITY;
    for (int c = threadIdx.x; c < C; c += kT) top = fmaxf(top, load_elem<T>(p, c * inner));
    top = block_all(top, buf, OpMax());
    const float m = top == -INFINITY ? 0.f : top;
    float all = 0.f, spare = 0.f;
    for (int c = threadIdx.x; c < C; c += kT) {
        const float e = expf((load_elem<T>(p, c * inner) - m) * inv_t);
        bool listed = false;
        for (int s = 0; s < k; ++s) listed |= t.idx[s] == c;
        all += e;
        spare += listed ? 0.f : e;
    }
    all = block_all(all, buf, OpAdd());
    spare = block_all(spare, buf, OpAdd());
    if (threadIdx.x == 0) {
        const float ls = all == 0.f ? 0.f : logf(all), lr = logf(spare);
        float loss = t.pr != 0.f ? t.pr * (t.logpr - (lr - ls)) : 0.f;
        for (int s = 0; s < k; ++s)
            if (t.idx[s] >= 0 && t.idx[s] < C && t.p[s] != 0.f)
                loss += t.p[s] * (t.logp[s] - ((load_elem<T>(p, t.idx[s] * inner) - m) * inv_t - ls));
        row_loss[row] = t.bad ? NAN : temp * temp * loss;
        stats[row] = make_float4(t.bad ? NAN : m, ls, spare == 0.f ? 0.f : lr, spare == 0.f ? 2.f : 1.f);
    }
}

// loss[0] = sum or mean of the rows that count, loss[1] = the factor of the gradient (1 / their number for the mean)
__global__ void __launch_bounds__(kT) distill_reduce_kernel(const float4* __restrict__ stats, const float* __restrict__ row_loss, long rows,
                                                            int mean, float* __restrict__ loss) {
    __shared__ double sums[kT], counts[kT];
    double s = 0.0, n = 0.0;
    for (long r = threadIdx.x; r < rows; r += kT)
        if (stats[r].w != 0.f) s += (double)row_loss[r], n += 1.0;
    sums[threadIdx.x] = s;
    counts[threadIdx.x] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kT; ++i) s += sums[i], n += counts[i];
        const double f = mean ? 1.0 / (n > 0.0 ? n : 1.0) : 1.0;
        loss[0] = (float)(s * f);
        loss[1] = (float)f;
    }
}

template <typename T>
__global__ void __launch_bounds__(kT) distill_bwd_kernel(const T* __restrict__ z, long ld, int C, long inner, int k,
                                                         const float* __restrict__ values, const int* __restrict__ indices,
                                                         const float* __restrict__ rest, float temp, float inv_t,
                                                         const float4* __restrict__ stats, const float* __restrict__ factor,
                                                         const float* __restrict__ g, int g_rows, T* __restrict__ dz) {
    __shared__ Teacher t;
    const long row = blockIdx.x, o = row / inner, i = row % inner;
    const float4 st = stats[row];
    T* d = dz + o * C * inner + i;
    if (st.w == 0.f) {
        for (int c = threadIdx.x; c < C; c += kT) store_elem<T>(d, c * inner, 0.f);
        return;
    }
    teacher_row(t, values, indices, rest, row, o, i, inner, k, C, inv_t);
    const T* p = z + o * ld + i;
    const float gs = g[g_rows ? row : 0] * (factor != nullptr ? factor[1] : 1.f) * temp;
    const float outside = (st.w == 2.f ? 0.f : expf(st.z - st.y)) - t.pr;
    for (int c = threadIdx.x; c < C; c += kT) {
        const float a = (load_elem<T>(p, c * inner) - st.x) * inv_t;
        bool listed = false;
        float sum = 0.f;
        for (int s = 0; s < k; ++s)
            if (t.idx[s] == c) listed = true, sum += t.p[s];
        store_elem<T>(d, c * inner, gs * (listed ? expf(a - st.y) - sum : expf(a - st.z) * outside));
    }
}

}  // namespace

#define ST(s) reinterpret_cast<hipStream_t>(s)

static bool layout_ok(long outer, int classes, long inner, long ld) {
    return outer >= 0 && classes > 0 && inner > 0 && (outer <= 1 || ld >= classes * inner) && (inner == 1 || ld == classes * inner) &&
           (outer == 0 || inner <= 0xffffffL / outer);  // a grid holds fewer than 2^32 threads
}

extern "C" int msfwsi_top_logits(int dtype, const void* x, long ld, long outer, int classes, long inner, int k, float inv_t, float* values,
                                 int* indices, float* rest, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && layout_ok(outer, classes, inner, ld) && k > 0 && k <= kMaxK && k <= classes && inv_t > 0.f);
    if (outer == 0) return MSFWSI_OK;
    MSFWSI_CHECK_ARG(x && values && indices && rest);
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL(top_logits_kernel<T>, dim3((unsigned)(outer * inner)), dim3(kT), 0, ST(stream), (const T*)x, ld,
                                            classes, inner, k, inv_t, values, indices, rest));
    return msfwsi_launch_status();
}

extern "C" int msfwsi_distill_fwd(int dtype, const void* z, long ld, long outer, int classes, long inner, int k, const float* values,
                                  const int* indices, const float* rest, const unsigned char* mask, float temperature, int mean, float* stats,
                                  float* row_loss, float* loss, double* partials, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && layout_ok(outer, classes, inner, ld) && k > 0 && k <= kMaxK && temperature > 0.f);
    MSFWSI_CHECK_ARG(loss && partials);
    if (outer > 0) {
        MSFWSI_CHECK_ARG(z && values && indices && stats && row_loss);
        MSFWSI_WITH_T(dtype, hipLaunchKernelGGL(distill_fwd_kernel<T>, dim3((unsigned)(outer * inner)), dim3(kT), 0, ST(stream), (const T*)z, ld,
                                                classes, inner, k, values, indices, rest, mask, temperature, 1.f / temperature, (float4*)stats,
                                                row_loss));
        const int rc = msfwsi_launch_status();
        if (rc != MSFWSI_OK) return rc;
    }
    hipLaunchKernelGGL(distill_reduce_kernel, dim3(1), dim3(kT), 0, ST(stream), (const float4*)stats, row_loss, outer * inner, mean, loss);
    return msfwsi_launch_status();
}

extern "C" int msfwsi_distill_bwd(int dtype, const void* z, long ld, long outer, int classes, long inner, int k, const float* values,
                                  const int* indices, const float* rest, float temperature, const float* stats, const float* factor,
                                  const float* g, int g_rows, void* dz, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && layout_ok(outer, classes, inner, ld) && k > 0 && k <= kMaxK && temperature > 0.f);
    if (outer == 0) return MSFWSI_OK;
    MSFWSI_CHECK_ARG(z && values && indices && stats && g && dz);
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL(distill_bwd_kernel<T>, dim3((unsigned)(outer * inner)), dim3(kT), 0, ST(stream), (const T*)z, ld,
                                            classes, inner, k, values, indices, rest, temperature, 1.f / temperature, (const float4*)stats,
                                            factor, g, g_rows, (T*)dz));
    return msfwsi_launch_status();
}
