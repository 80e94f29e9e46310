// Distillation from a teacher's largest logits: their selection, and the loss of a student against them with its gradient.
//
// Logits lie as [outer][classes][inner] (inner = 1: rows of logits, which may be `ld` elements apart; inner > 1: maps
// [N, C, H * W]); a "row" is one (outer, inner) position.
//
// Selection: the k largest logits of a row in descending order, equal ones by ascending index, NaN above every number; and
//   rest = log sum over the OTHERS of exp(logit / T)          (-inf when nothing is left, +inf when one of them is +inf)
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

#include <type_traits>

namespace {

constexpr int kT = 256;
constexpr int kMaxK = 64;        // = the lanes of a wave: lane i holds entry i of a teacher's list
constexpr int kMaxParts = 8192;  // workgroups of the forward at most; each leaves one (sum, count) pair
constexpr int kSeg = 65536;      // classes whose list membership is held as bits at a time
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// 2^x and log2 x as the hardware has them (1 ulp; results below 2^-126 are flushed: sums are taken relative to their largest term)
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }

// fp32 -> int of the same order; -0 equals +0, every NaN is the largest
__device__ __forceinline__ int order_of(float x) {
    if (x != x) return 0x7fffffff;
    const int b = (int)__float_as_uint(x + 0.f);
    return b ^ ((b >> 31) & 0x7fffffff);
}
constexpr int kNothing = (int)0x80000000;  // the order of an empty slot, below every number's
__device__ __forceinline__ float value_of(int order) {
    if (order == kNothing) return -INFINITY;
    return __uint_as_float((unsigned)(order ^ ((order >> 31) & 0x7fffffff)));
}
// (order, index) as one number: larger logits first, equal ones by ascending index; unique within a row
__device__ __forceinline__ long key_of(float x, int idx) { return ((long)order_of(x) << 32) | (unsigned)(0x7fffffff - idx); }
__device__ __forceinline__ int index_of(long key) { return 0x7fffffff - (int)(unsigned)key; }
constexpr long kNoKey = (long)0x8000000000000000L;

// sum of 2^((x - m) c) over some logits x: c = log2(e) / T, m the largest of them.  Nothing: m = -inf, s = 0; a NaN among them
// makes s NaN.  The difference is taken before the product, so logits far from zero keep their precision and a row of the
// type's lowest value does not overflow.  (c x - c m in one fma was no faster.)  With INF a logit of +inf is a term of 1 relative
// to itself and the logarithm of the sum +inf; without, a NaN (the loss has no softmax there, and its kernels no registers to spare).
struct Sum {
    float m, s;
};
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.f : m; }
template <bool INF>
__device__ __forceinline__ float term(float x, float ref, float c) {
    return INF && x == ref ? 1.f : exp2_((x - ref) * c);
}
template <bool INF>
__device__ __forceinline__ Sum join(Sum a, Sum b, float c) {
    const float m = fmaxf(a.m, b.m), ref = finite_ref(m);
    return {m, a.s * term<INF>(a.m, ref, c) + b.s * term<INF>(b.m, ref, c)};
}
__device__ __forceinline__ Sum one(float x) { return {x, x == -INFINITY ? 0.f : 1.f}; }
// The same taken by one lane over any number of logits, 32 at a time: the sums of 32 are added with what the additions before lost
// put back (compensated), and the reference moves only where a logit exceeds it by more than kRaise powers of two, so the error
// is that of 32 additions whatever the number (70001 equal logits behind one a little larger, added one by one: the logarithm 6.5e-4 off).
constexpr float kRaise = 1.f;
constexpr int kAtOnce = 32;
struct LongSum {
    float ref = -INFINITY, total = 0.f, lost = 0.f;
    __device__ __forceinline__ bool raises(float x, float c) const { return (x - ref) * c > kRaise; }
    __device__ __forceinline__ float raise(float to, float c) {  // the factor, for what has not been added yet
        const float f = exp2_((ref - to) * c);
        total *= f;
        lost *= f;
        ref = to;
        return f;
    }
    __device__ __forceinline__ void add(float part) {
        const float y = part - lost, t = total + y;
        lost = (t - total) - y;
        total = t;
    }
};
__device__ __forceinline__ float log_of(Sum v, float inv_t) { return v.s == 0.f ? -INFINITY : v.m * inv_t + log2_(v.s) * kLn2; }
template <bool INF>
__device__ __forceinline__ Sum wave_join(Sum v, float c) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = join<INF>(v, {__shfl_xor(v.m, off, 64), __shfl_xor(v.s, off, 64)}, c);
    return v;
}
// over the workgroup; every thread has the result
template <int NT, bool INF>
__device__ __forceinline__ Sum block_join(Sum v, Sum* buf, float c) {
    v = wave_join<INF>(v, c);
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
        __syncthreads();
        v = buf[0];
        for (int i = 1; i < NT / 64; ++i) v = join<INF>(v, buf[i], c);
        __syncthreads();
    }
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float o = __shfl_xor(v, off, 64);
        v = v != v || o <= v ? v : o;  // NaN stays
    }
    return v;
}

// 16 bytes of a row at any alignment; elements past the row are -inf
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Unaligned16 {
    unsigned x, y, z, w;
};
template <typename T>
__device__ __forceinline__ uint4 whole_chunk(const T* __restrict__ p, int c) {
    const Unaligned16<T> u = *reinterpret_cast<const Unaligned16<T>*>(p + c);
    return make_uint4(u.x, u.y, u.z, u.w);
}
// the same for a row that is read once: not kept in the caches (155 -> 149 us at 4096 x 65536)
template <typename T>
__device__ __forceinline__ uint4 passing_chunk(const T* __restrict__ p, int c) {
    typedef __attribute__((ext_vector_type(4), aligned(2))) unsigned u32x4_any;
    const u32x4_any u = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p + c));
    return make_uint4(u.x, u.y, u.z, u.w);
}
template <typename T>
__device__ __forceinline__ uint4 load_chunk(const T* __restrict__ p, int c, int n) {
    constexpr int VEC = ElemTraits<T>::VEC;
    if (c + VEC <= n) return whole_chunk<T>(p, c);
    float f[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = c + e < n ? load_elem<T>(p, c + e) : -INFINITY;
    return pack16<T>(f);
}
// keeps hipcc from carrying the unpacked forms of a register chunk (2x its size, more with their keys) from one walk to the next
__device__ __forceinline__ void unknown(uint4& v) { asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w)); }
template <typename T>
__device__ __forceinline__ void store_chunk(T* __restrict__ p, int c, int n, const float* f) {
    constexpr int VEC = ElemTraits<T>::VEC;
    if (c + VEC <= n) {
        const uint4 v = pack16<T>(f);
        *reinterpret_cast<Unaligned16<T>*>(p + c) = {v.x, v.y, v.z, v.w};
        return;
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e)
        if (c + e < n) store_elem<T>(p, c + e, f[e]);
}

// ---------------------------------------------------------------------------------------------------------------------
// Selection, rows of adjacent classes.  A workgroup holds one segment of a row in registers (read once): NT threads x NCH
// chunks of 16 bytes.  The k-th largest of the NT threads' maxima is a lower bound of the k-th largest element, found by
// one wave bit by bit with ballots.  Chunks that hold anything not below it -- barely more than k unless large logits crowd
// into few threads or tie -- go to a queue, whose elements the threads then look at one by one (nearly every wave meets such a
// chunk at nearly every step: looking at them in place cost all lanes the walk twice over, 166 us instead of 149); what is
// not below the bound goes into a list and is ranked by counting.  Everything else is summed for `rest`, each thread its own and the
// list's surplus once it is in order: the lists fill in any order, no sum depends on it.
// 4096 rows of 65536 bf16, k = 32: 132 us, 4.1 TB/s, the vector units busy throughout; 4 such rows of fp32 8 us.
// A queue or list that runs over (long ties, a masked-out segment) sends the segment through k rounds of a plain maximum instead.
// Rows longer than a segment leave their segments' lists and sums to a merge.
// DEEP: a list of more than 16 from a row that one wave takes.  The k-th of only 64 maxima would leave most of the row for candidates,
// so the maxima are those of single chunks (65536 rows of 1000 bf16, k = 64: 186 us; 726 with one maximum a thread).
// ---------------------------------------------------------------------------------------------------------------------
// Seven waves a SIMD of a segment's 256 threads leave 72 registers each; fp16 needs a few more and spilled: six (4096 x 65536 at
// k = 32: 156 -> 147 us).
template <typename T, int NT, int NCH, bool DEEP>
__global__ void __launch_bounds__(NT, NT == 256 ? (__is_same(T, _Float16) ? 6 : 7) : DEEP ? 4 : 5) top_segment_kernel(const T* __restrict__ x, long ld, int C, int nseg, int k, float inv_t,
                                                         float* __restrict__ values, int* __restrict__ indices, float* __restrict__ rest,
                                                         long* __restrict__ part_keys, Sum* __restrict__ part_sums) {
    constexpr int VEC = ElemTraits<T>::VEC;
    constexpr int GROUPS = DEEP ? NT * NCH : NT;                        // maxima that the bound is found among
    constexpr int kQueue = NT == 256 ? 256 : DEEP ? 128 : 64;           // chunks with candidates
    constexpr int kCand = NT == 256 || DEEP ? 512 : 128;                // candidates that are ranked at once
    constexpr int kShared = kQueue * 16 > kCand * 8 ? kQueue * 16 : kCand * 8;
    __shared__ long cand[kCand];
    __shared__ __attribute__((aligned(16))) char shared_[kShared];
    __shared__ int queue_at[kQueue];
    __shared__ int maxima[GROUPS];
    uint4* queue = reinterpret_cast<uint4*>(shared_);
    long* sorted = reinterpret_cast<long*>(shared_);  // once the queue has been read
    __shared__ Sum buf[NT / 64];
    __shared__ long lbuf[NT / 64];
    __shared__ int count, queued, bound;
    const int t = threadIdx.x;
    const long row = blockIdx.x / nseg;
    const int seg = (int)(blockIdx.x % nseg), c0 = seg * (NT * NCH * VEC), n = min(C - c0, NT * NCH * VEC), want = min(k, n);
    const T* p = x + row * ld + c0;
    const float c = inv_t * kLog2e;
    long* keys_out = part_keys + (long)blockIdx.x * k;

    uint4 raw[NCH];
    float f[VEC], top = -INFINITY;
    if (n == NT * NCH * VEC) {
#pragma unroll
        for (int j = 0; j < NCH; ++j) raw[j] = passing_chunk<T>(p, (j * NT + t) * VEC);
    } else {
#pragma unroll
        for (int j = 0; j < NCH; ++j) raw[j] = load_chunk<T>(p, (j * NT + t) * VEC, n);
    }
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        unpack16<T>(raw[j], f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) top = fmaxf(top, f[e]);
        if constexpr (DEEP) maxima[j * NT + t] = order_of(top), top = -INFINITY;
    }
    if constexpr (!DEEP) maxima[t] = order_of(top);
    if (t == 0) count = queued = 0;
    __syncthreads();
    if (t < 64) {
        int m[GROUPS / 64];
#pragma unroll
        for (int i = 0; i < GROUPS / 64; ++i) m[i] = maxima[i * 64 + t];
        // the 20 highest bits: 16-bit types whole, fp32 to 2^-11 of its value; a lower bound is all that is needed
        int b = kNothing;
#pragma unroll 1
        for (int bit = 31; bit >= 12; --bit) {
            const int raised = bit == 31 ? 0 : b | (1 << bit);
            int above = 0;
#pragma unroll
            for (int i = 0; i < GROUPS / 64; ++i) above += __popcll(__ballot(m[i] >= raised));
            if (above >= k) b = raised;
        }
        if (t == 0) bound = b;
    }
    __syncthreads();
    const int b = bound;
    // an order below that of -inf (too few maxima, or cut-off bits) leaves nothing out
    const float lim = b <= (int)0x807fffff ? -INFINITY : value_of(b);
    const float shift = -finite_ref(lim * c);  // c x - c lim in one fma: `rest` itself has no finer step than c lim's
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        unknown(raw[j]);
        unpack16<T>(raw[j], f);
        float high = f[0], part = 0.f;
#pragma unroll
        for (int e = 1; e < VEC; ++e) high = fmaxf(high, f[e]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float x2 = exp2_(fmaf(f[e], c, shift));
            part += f[e] >= lim ? 0.f : x2;
        }
        // a row of fewer than k chunks has no bound: its own chunks go in, those past its end do not
        const bool queue_it = !(high < lim) && (NT == 256 || (j * NT + t) * VEC < n);
        s += part;
        if (queue_it) {
            const int slot = atomicAdd(&queued, 1);
            if (slot < kQueue) queue[slot] = raw[j], queue_at[slot] = (j * NT + t) * VEC;
        }
    }
    __syncthreads();
    const int chunks = queued;
    if (chunks <= kQueue)
        for (int i = t; i < chunks * VEC; i += NT) {
            const int at = queue_at[i / VEC] + i % VEC;
            const float v = load_elem<T>(reinterpret_cast<const T*>(queue), i);
            if (at >= n) continue;
            if (!(v < lim)) {
                const int slot = atomicAdd(&count, 1);
                if (slot < kCand) cand[slot] = key_of(v, c0 + at);
            }
        }
    const Sum below = block_join<NT, false>({s == 0.f ? -INFINITY : finite_ref(lim), s}, buf, c);
    __syncthreads();
    const int got = count;
    Sum left = {-INFINITY, 0.f};
    // The list decides when it holds every candidate.  The sum decides unless a NaN went by in it, or it is so small against its
    // reference that the terms flushed from it count: up to 16384, each below 2^-126, are under 2^-24 of a sum of 2^-88
    if (chunks <= kQueue && got <= kCand && (got >= n || below.s >= 0x1p-88f)) {
        for (int i = t; i < got; i += NT) {
            const long key = cand[i];
            int rank = 0;
            for (int q = 0; q < got; ++q) rank += cand[q] > key;
            sorted[rank] = key;
        }
        __syncthreads();
        for (int i = t; i < got; i += NT) {
            const long key = sorted[i];
            if (i >= want) {
                left = join<false>(left, one(value_of((int)(key >> 32))), c);
            } else if (nseg == 1) {
                values[row * k + i] = value_of((int)(key >> 32));
                indices[row * k + i] = index_of(key);
            } else {
                keys_out[i] = key;
            }
        }
        left = block_join<NT, false>(left, buf, c);
        if (got < n) left = join<false>(below, left, c);  // else there is nothing below, and a NaN in that sum is a candidate
        // +inf left over comes first of the surplus, behind a NaN alone (join<true> in these sums: 132 -> 137 us at 4096 x 65536)
        if (left.m == INFINITY && value_of((int)(sorted[want] >> 32)) == INFINITY) left.s = 1.f;
    } else {
        long last = 0x7fffffffffffffffL;
        for (int r = 0; r < want; ++r) {
            long best = kNoKey;
            int mine = t;
            asm volatile("" : "+v"(mine));  // its elements' keys are formed anew in every round
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                unknown(raw[j]);
                unpack16<T>(raw[j], f);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int at = (j * NT + mine) * VEC + e;
                    const long key = key_of(f[e], c0 + at);
                    if (at < n && key < last && key > best) best = key;
                }
            }
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) {
                const long o = __shfl_xor(best, off, 64);
                best = o > best ? o : best;
            }
            if constexpr (NT > 64) {
                if ((t & 63) == 0) lbuf[t >> 6] = best;
                __syncthreads();
                best = lbuf[0];
                for (int i = 1; i < NT / 64; ++i) best = lbuf[i] > best ? lbuf[i] : best;
                __syncthreads();
            }
            last = best;
            if (t == 0) {
                if (nseg == 1) {
                    values[row * k + r] = value_of((int)(last >> 32));
                    indices[row * k + r] = index_of(last);
                } else {
                    keys_out[r] = last;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            unknown(raw[j]);
            unpack16<T>(raw[j], f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int at = (j * NT + t) * VEC + e;
                if (at < n && key_of(f[e], c0 + at) < last) left = join<true>(left, one(f[e]), c);
            }
        }
        left = block_join<NT, true>(left, buf, c);
    }
    if (t == 0) {
        if (nseg == 1) rest[row] = log_of(left, inv_t);
        else part_sums[blockIdx.x] = left;
    }
    if (nseg > 1)
        for (int r = want + t; r < k; r += NT) keys_out[r] = kNoKey;
}

// The segments' lists of a row become one: every entry's rank is counted (33 us as rounds over the lists' heads, 15 so, at
// 4096 rows of 4 x 32); what is not among the k joins `rest`.
constexpr int kMergeHeld = 2048;
__global__ void __launch_bounds__(kT) top_merge_kernel(const long* __restrict__ part_keys, const Sum* __restrict__ part_sums, int nseg, int k,
                                                       float inv_t, float* __restrict__ values, int* __restrict__ indices,
                                                       float* __restrict__ rest) {
    extern __shared__ long held[];
    __shared__ Sum buf[kT / 64];
    const int t = threadIdx.x, n = nseg * k;
    const long row = blockIdx.x;
    const long* keys = part_keys + row * n;
    const float c = inv_t * kLog2e;
    for (int i = t; i < n; i += kT) held[i] = keys[i];
    __syncthreads();
    Sum sum = {-INFINITY, 0.f};
    for (int i = t; i < nseg; i += kT) sum = join<true>(sum, part_sums[row * nseg + i], c);
    for (int i = t; i < n; i += kT) {
        const long key = held[i];
        if (key == kNoKey) continue;
        int rank = 0;
#pragma unroll 8
        for (int q = 0; q < n; ++q) rank += held[q] > key;
        if (rank < k) {
            values[row * k + rank] = value_of((int)(key >> 32));
            indices[row * k + rank] = index_of(key);
        } else {
            sum = join<true>(sum, one(value_of((int)(key >> 32))), c);
        }
    }
    sum = block_join<kT, true>(sum, buf, c);
    if (t == 0) rest[row] = log_of(sum, inv_t);
}
// The same for more entries than are worth counting: one wave per row, k rounds over the heads of the sorted lists.
__global__ void __launch_bounds__(64) top_merge_long_kernel(const long* __restrict__ part_keys, const Sum* __restrict__ part_sums, int nseg,
                                                            int k, float inv_t, float* __restrict__ values, int* __restrict__ indices,
                                                            float* __restrict__ rest) {
    extern __shared__ int head[];  // entry i belongs to lane i % 64 alone
    const int l = threadIdx.x;
    const long row = blockIdx.x;
    const long* keys = part_keys + row * nseg * k;
    const float c = inv_t * kLog2e;
    long mine = kNoKey;
    int from = -1;
    for (int i = l; i < nseg; i += 64) {
        head[i] = 0;
        if (keys[(long)i * k] > mine) mine = keys[(long)i * k], from = i;
    }
    for (int r = 0; r < k; ++r) {
        long best = mine;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const long o = __shfl_xor(best, off, 64);
            best = o > best ? o : best;
        }
        if (mine == best && from >= 0) {
            values[row * k + r] = value_of((int)(best >> 32));
            indices[row * k + r] = index_of(best);
            head[from]++;
            mine = kNoKey;
            from = -1;
            for (int i = l; i < nseg; i += 64)
                if (head[i] < k && keys[(long)i * k + head[i]] > mine) mine = keys[(long)i * k + head[i]], from = i;
        }
    }
    Sum sum = {-INFINITY, 0.f};
    for (int i = l; i < nseg; i += 64) {
        sum = join<true>(sum, part_sums[row * nseg + i], c);
        for (int r = head[i]; r < k; ++r) {
            const long key = keys[(long)i * k + r];
            if (key != kNoKey) sum = join<true>(sum, one(value_of((int)(key >> 32))), c);
        }
    }
    sum = wave_join<true>(sum, c);
    if (l == 0) rest[row] = log_of(sum, inv_t);
}

// ---------------------------------------------------------------------------------------------------------------------
// Selection, one thread per row: maps (neighbouring threads, neighbouring positions) and rows of a few classes.  The list is
// kept sorted in registers; every class throws one value out of it (itself, a displaced one or an empty slot), which goes to
// the running sum for `rest`, so the logits are read once.  KM places: 4, 16 or 64 (16 maps of 21 x 256 x 256 bf16: k = 4 in 4 / 16 / 64
// places 30 / 58 / 268 us, k = 16 in 16 / 64 63 / 272).
// ---------------------------------------------------------------------------------------------------------------------
// 16-bit logits: order and index fit one int (up to 65536 classes), and a step of the insertion is a max and a min.
template <typename T>
__device__ __forceinline__ int order16(T x);
template <>
__device__ __forceinline__ int order16<__bf16>(__bf16 x) { return order_of((float)x) >> 16; }
template <>
__device__ __forceinline__ int order16<_Float16>(_Float16 x) {
    if (x != x) return 0x7fff;
    const int b = __builtin_bit_cast(short, (_Float16)(x + (_Float16)0.f));
    return b ^ ((b >> 15) & 0x7fff);
}
template <typename T>
__device__ __forceinline__ float value16(int order);
template <>
__device__ __forceinline__ float value16<__bf16>(int order) { return __uint_as_float((unsigned)(order ^ ((order >> 15) & 0x7fff)) << 16); }
template <>
__device__ __forceinline__ float value16<_Float16>(int order) {
    return (float)__builtin_bit_cast(_Float16, (short)(order ^ ((order >> 15) & 0x7fff)));
}
template <typename T, int KM, bool SMALL>
__global__ void __launch_bounds__(kT) top_thread_kernel(const T* __restrict__ x, long ld, int C, long inner, long rows, int k, float inv_t,
                                                        float* __restrict__ values, int* __restrict__ indices, float* __restrict__ rest) {
    const float c = inv_t * kLog2e;
    const long row = blockIdx.x * (long)kT + threadIdx.x;
    if (row >= rows) return;
    const long o = (unsigned)row / (unsigned)inner, i = row - o * inner;  // rows fit 31 bits
    const T* p = x + o * ld + i;
    int v[KM], at[SMALL ? 1 : KM];
#pragma unroll
    for (int s = 0; s < KM; ++s) v[s] = kNothing;
    if constexpr (!SMALL) {
#pragma unroll
        for (int s = 0; s < KM; ++s) at[s] = 0;
    }
    LongSum sum;
    float part = 0.f;
    bool infinite = false;
    // class j's logit goes in, what it throws out of the list comes back
    auto insert = [&](T x_, int j) {
        if constexpr (SMALL) {
            int a = order16<T>(x_) << 16 | (0xffff - j);
#pragma unroll
            for (int s = 0; s < KM; ++s)
                if (s < k) {
                    const int low = min(v[s], a);
                    v[s] = max(v[s], a);
                    a = low;
                }
            return a == kNothing ? -INFINITY : value16<T>(a >> 16);
        } else {
            int a = order_of((float)x_), ai = j;
            bool in = false;
#pragma unroll
            for (int s = 0; s < KM; ++s)
                if (s < k) {
                    const int ov = v[s], oi = at[s];
                    in = in || a > ov;
                    v[s] = in ? a : ov;
                    at[s] = in ? ai : oi;
                    a = in ? ov : a;
                    ai = in ? oi : ai;
                }
            return value_of(a);
        }
    };
    auto sum_up = [&](float (&out)[4]) {
        float high = fmaxf(fmaxf(out[0], out[1]), fmaxf(out[2], out[3]));
        if (sum.raises(high, c)) {
            if (high == INFINITY) {  // kept apart: the sum has no term for it
                infinite = true;
                high = -INFINITY;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (out[u] == INFINITY) out[u] = -INFINITY;
                    high = fmaxf(high, out[u]);
                }
            }
            if (sum.raises(high, c)) part *= sum.raise(high, c);
        }
        const float ref = finite_ref(sum.ref);
#pragma unroll
        for (int u = 0; u < 4; ++u) part += exp2_((out[u] - ref) * c);
    };
    int j = 0;
    for (; j + 4 <= C; j += 4) {
        T raw[4];
        float out[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) raw[u] = p[(j + u) * inner];
#pragma unroll
        for (int u = 0; u < 4; ++u) out[u] = insert(raw[u], j + u);
        sum_up(out);
        if ((j & (kAtOnce - 1)) == kAtOnce - 4) {
            sum.add(part);
            part = 0.f;
        }
    }
    for (; j < C; ++j) {
        float out[4] = {insert(p[j * inner], j), -INFINITY, -INFINITY, -INFINITY};
        sum_up(out);
    }
    sum.add(part);
#pragma unroll
    for (int s = 0; s < KM; ++s)
        if (s < k) {
            if constexpr (SMALL) values[(o * k + s) * inner + i] = value16<T>(v[s] >> 16);
            else values[(o * k + s) * inner + i] = value_of(v[s]);
            indices[(o * k + s) * inner + i] = SMALL ? 0xffff - (v[s] & 0xffff) : at[s];
        }
    rest[row] = infinite && sum.total == sum.total ? INFINITY : log_of({sum.ref, sum.total}, inv_t);
}

// ---------------------------------------------------------------------------------------------------------------------
// The loss.  What the backward keeps of a row, in four floats: m and s of the sum over all classes (struct Sum), and the
// same, mt and st, over the unlisted ones.  Two maxima, because the unlisted classes may lie so far below the
// listed ones that their sum relative to m would vanish.  s = -1 marks a row that does not count.  The sums themselves and not their
// logarithms: log2 s of 65536 classes has a step of 2^-20, and as a part of the exponent it put every q of a row off by up to
// 6 2^-24; a product with 1 / s is off by 2 2^-24.
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float4 row_stats(Sum unlisted, Sum all) {
    const float m = finite_ref(all.m);
    return make_float4(m, all.s, unlisted.m == -INFINITY ? m : unlisted.m, unlisted.s);
}
__device__ __forceinline__ bool row_counts(const float4& st) { return st.y != -1.f; }
__device__ __forceinline__ float log2_sum(float s) { return s == 0.f ? 0.f : log2_(s); }
// 1 / s, 1 ulp; 0 of an empty sum, so that a softmax over nothing is zero
__device__ __forceinline__ float part_of(float s) { return s == 0.f ? 0.f : __builtin_amdgcn_rcpf(s); }

// (sum, count) of the rows that count, one pair per workgroup, joined in a fixed order
template <int NT>
__device__ __forceinline__ void leave_part(double s, double n, double* __restrict__ parts) {
    __shared__ double buf[2][NT / 64];
    s = wave_sum_d(s);
    n = wave_sum_d(n);
    if ((threadIdx.x & 63) == 0) buf[0][threadIdx.x >> 6] = s, buf[1][threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < NT / 64; ++i) s += buf[0][i], n += buf[1][i];
        parts[2 * blockIdx.x] = s;
        parts[2 * blockIdx.x + 1] = n;
    }
}
// loss = sum or mean of the rows that count, factor = that of the gradient (1 / their number for the mean)
constexpr int kFinish = 1024;
__global__ void __launch_bounds__(kFinish) distill_finish_kernel(const double* __restrict__ parts, int n, int mean, float* __restrict__ loss,
                                                            float* __restrict__ factor) {
    __shared__ double sums[kFinish / 64], counts[kFinish / 64];
    double s = 0.0, m = 0.0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) s += parts[2 * i], m += parts[2 * i + 1];
    s = wave_sum_d(s);
    m = wave_sum_d(m);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s, counts[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < (int)blockDim.x / 64; ++i) s += sums[i], m += counts[i];
        const double f = mean ? 1.0 / (m > 0.0 ? m : 1.0) : 1.0;
        *loss = (float)(s * f);
        *factor = (float)f;
    }
}

// Rows of adjacent classes, a workgroup per row (64 threads for short rows: one wave, no barriers between waves).  Lane i of
// every wave holds entry i of the teacher's list; the classes it lists are a bit set in LDS, one byte (fp32: half a byte) per
// 16-byte chunk.  One walk over the row sums the unlisted classes; the listed ones are gathered.  Bound by reading the row and, near
// that, by an exponential per class: 4096 rows of 65536 bf16 136 us, 3.9 TB/s.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) distill_fwd_kernel(const T* __restrict__ z, long ld, int C, long rows, int k,
                                                         const float* __restrict__ values, const int* __restrict__ indices,
                                                         const float* __restrict__ rest, const unsigned char* __restrict__ mask, float temp,
                                                         float inv_t, float4* __restrict__ stats, float* __restrict__ row_loss,
                                                         double* __restrict__ parts) {
    constexpr int VEC = ElemTraits<T>::VEC;
    constexpr int SEG = NT == 64 ? 4096 : kSeg;
    constexpr int U = 4;  // chunks in flight per thread
    __shared__ unsigned bits[SEG / 32];
    __shared__ Sum buf[NT / 64];
    const int t = threadIdx.x, lane = t & 63;
    const float c = inv_t * kLog2e;
    for (int i = t; i < SEG / 32; i += NT) bits[i] = 0;
    double lsum = 0.0, lcount = 0.0;
    for (long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* p = z + row * ld;
        const int idx = lane < k ? indices[row * k + lane] : -1;
        const float v = idx >= 0 ? values[row * k + lane] : -INFINITY, r = rest != nullptr ? rest[row] * temp : -INFINITY;
        const float vtop = wave_max(v != v || r <= v ? v : r);
        if (vtop == -INFINITY || (mask != nullptr && mask[row] == 0)) {
            if (t == 0) {
                stats[row] = make_float4(0.f, -1.f, 0.f, 0.f);
                if (row_loss != nullptr) row_loss[row] = 0.f;
            }
            continue;
        }
        Sum sum = {-INFINITY, 0.f};
        for (int s0 = 0; s0 < C; s0 += SEG) {
            const int n = min(C - s0, SEG);
            const bool here = t < 64 && idx >= s0 && idx - s0 < n;
            __syncthreads();
            if (here) atomicOr(&bits[(idx - s0) >> 5], 1u << ((idx - s0) & 31));
            __syncthreads();
            auto add = [&](const uint4* raw, int a, auto count_) {  // chunks of this thread from `a` on
                constexpr int N = decltype(count_)::value;
                float f[N][VEC];
                float top = -INFINITY;
#pragma unroll
                for (int u = 0; u < N; ++u) {
                    const int at = a + (u * NT + t) * VEC;
                    unpack16<T>(raw[u], f[u]);
                    const unsigned w = at < n ? (bits[at >> 5] >> (at & 31)) & ((1u << VEC) - 1u) : 0u;
                    if (w) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) f[u][e] = (w >> e) & 1u ? -INFINITY : f[u][e];
                    }
#pragma unroll
                    for (int e = 0; e < VEC; ++e) top = fmaxf(top, f[u][e]);
                }
                const float m = fmaxf(sum.m, top), ref = finite_ref(m);
                float s = 0.f;  // a turn's terms by themselves: the long row's sum takes one addition for them
#pragma unroll
                for (int u = 0; u < N; ++u)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) s += exp2_((f[u][e] - ref) * c);
                sum = {m, fmaf(sum.s, exp2_((sum.m - ref) * c), s)};
            };
            // whole turns of U chunks a thread, loaded without a test each (a load behind a branch of its own is waited for there)
            // and one turn ahead; then the rest chunk by chunk
            constexpr int TURN = U * NT * VEC;
            int a = 0;
            if (n >= TURN) {
                uint4 raw[U], next[U];
#pragma unroll
                for (int u = 0; u < U; ++u) raw[u] = whole_chunk<T>(p + s0, (u * NT + t) * VEC);
                for (; a + 2 * TURN <= n; a += TURN) {
#pragma unroll
                    for (int u = 0; u < U; ++u) next[u] = whole_chunk<T>(p + s0, a + TURN + (u * NT + t) * VEC);
                    add(raw, a, std::integral_constant<int, U>());
#pragma unroll
                    for (int u = 0; u < U; ++u) raw[u] = next[u];
                }
                add(raw, a, std::integral_constant<int, U>());
                a += TURN;
            }
            for (; a < n; a += NT * VEC) {
                const uint4 raw = load_chunk<T>(p + s0, a + t * VEC, n);  // past the row: all -inf
                add(&raw, a, std::integral_constant<int, 1>());
            }
            __syncthreads();
            if (here) bits[(idx - s0) >> 5] = 0;
        }
        const Sum unlisted = block_join<NT, false>(sum, buf, c);
        if (t < 64) {
            const bool valid = idx >= 0 && idx < C, bad = __any(idx >= C);
            const float zi = valid ? load_elem<T>(p, idx) : -INFINITY;
            bool first = valid;
            for (int q = 0; q < k; ++q) {
                const int other = __shfl(idx, q, 64);  // by every lane: a lane that sits out cannot be read either
                first = first && (q >= lane || other != idx);
            }
            const float m = fmaxf(unlisted.m, wave_max(zi == zi ? zi : -INFINITY)), ref = finite_ref(m);
            const Sum all = {m, unlisted.s * exp2_((unlisted.m - ref) * c) + wave_sum(first ? exp2_((zi - ref) * c) : 0.f)};
            float4 st = row_stats(unlisted, all);
            if (bad) st.x = st.z = NAN;
            const float ls = log2_sum(st.y), lt = log2_sum(st.w);
            // teacher, in base-2 units relative to its largest entry
            const float lv = (v - vtop) * c, lr = (r - vtop) * c;
            const float L = log2_(wave_sum(lane < k ? exp2_(lv) : 0.f) + exp2_(lr));
            const float pi = lane < k ? exp2_(lv - L) : 0.f, pr = exp2_(lr - L);
            float term = pi != 0.f ? pi * ((lv - L) - ((zi - st.x) * c - ls)) : 0.f;
            if (lane == 0 && pr != 0.f) {
                const float lq = unlisted.s == 0.f ? -INFINITY : (st.z - st.x) * c + lt - ls;
                term += pr * ((lr - L) - lq);
            }
            const float loss = temp * temp * kLn2 * wave_sum(term);
            if (t == 0) {
                stats[row] = st;
                if (row_loss != nullptr) row_loss[row] = bad ? NAN : loss;
                lsum += (double)(bad ? NAN : loss);
                lcount += 1.0;
            }
        }
    }
    if (t == 0) parts[2 * blockIdx.x] = lsum, parts[2 * blockIdx.x + 1] = lcount;
}

// The unlisted form goes over the whole row; behind a barrier the lanes that hold the list put the listed classes right.  Bound by
// memory: 4096 rows of 65536 bf16 204 us, 5.3 TB/s read and written.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) distill_bwd_kernel(const T* __restrict__ z, long ld, int C, long rows, int k,
                                                         const float* __restrict__ values, const int* __restrict__ indices,
                                                         const float* __restrict__ rest, float temp, float inv_t,
                                                         const float4* __restrict__ stats, const float* __restrict__ factor,
                                                         const float* __restrict__ g, int g_rows, T* __restrict__ dz) {
    constexpr int VEC = ElemTraits<T>::VEC;
    constexpr int U = 4;
    const int t = threadIdx.x, lane = t & 63;
    const float c = inv_t * kLog2e;
    const long row = blockIdx.x;
    const T* p = z + row * ld;
    T* d = dz + row * (long)C;
    const float4 st = stats[row];
    if (!row_counts(st)) {
        float f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = 0.f;
        for (int a = t * VEC; a < C; a += NT * VEC) store_chunk<T>(d, a, C, f);
        return;
    }
    const int idx = lane < k ? indices[row * k + lane] : -1;
    const float v = idx >= 0 ? values[row * k + lane] : -INFINITY, r = rest != nullptr ? rest[row] * temp : -INFINITY;
    const float vtop = wave_max(v != v || r <= v ? v : r);
    const float wi = lane < k ? exp2_((v - vtop) * c) : 0.f, wr = exp2_((r - vtop) * c);
    const float share_of = part_of(wave_sum(wi) + wr), pi = wi * share_of, pr = wr * share_of;
    const float gs = g[g_rows ? row : 0] * (factor != nullptr ? *factor : 1.f) * temp;
    const float q_of = part_of(st.y), outside = gs * (exp2_((st.z - st.x) * c) * (st.w * q_of) - pr) * part_of(st.w);
    int a = 0;
    for (; a + U * NT * VEC <= C; a += U * NT * VEC) {
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = whole_chunk<T>(p, a + (u * NT + t) * VEC);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[VEC];
            unpack16<T>(raw[u], f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = outside * exp2_((f[e] - st.z) * c);
            store_chunk<T>(d, a + (u * NT + t) * VEC, C, f);
        }
    }
    for (a += t * VEC; a < C; a += NT * VEC) {
        float f[VEC];
        unpack16<T>(load_chunk<T>(p, a, C), f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = outside * exp2_((f[e] - st.z) * c);
        store_chunk<T>(d, a, C, f);
    }
    __syncthreads();
    if (t >= 64) return;
    float share = 0.f;  // of all entries with this lane's class
    for (int q = 0; q < k; ++q) {
        const int other = __shfl(idx, q, 64);
        const float po = __shfl(pi, q, 64);
        share += other == idx ? po : 0.f;
    }
    if (idx >= 0 && idx < C) store_elem<T>(d, idx, gs * (exp2_((load_elem<T>(p, idx) - st.x) * c) * q_of - share));
}

// One thread per row: maps, and rows of a few classes.  A class costs about 7 instructions: the listed ones are taken out of the
// sum by a bit each, their own logits are asked for early and handled apart.  32 maps of 21 x 256 x 256 fp32, k = 4: forward 100 us
// (2.9 TB/s; bound by latency and instructions: at 4 waves per SIMD the vector units are busy half the time), backward 106 us (4.4 TB/s).  KM > 0: lists of up to KM entries whose indices stay in registers;
// KM = 0: any length, read again where needed (the same maps, forward / with the gradient: k = 4 as KM 4 92 / 211 us, as 16 129 / 294, as
// 0 145 / 428; k = 16 as KM 16 305 / 626, as 0 693 / 2163).
template <int KM>
struct List {
    int idx[KM > 0 ? KM : 1];
    const int* ip;
    const float* vp;
    long inner;
    int k;
    __device__ __forceinline__ void open(const float* values, const int* indices, long o, long i, long inner_, int k_) {
        ip = indices + o * k_ * inner_ + i;
        vp = values + o * k_ * inner_ + i;
        inner = inner_;
        k = k_;
        if constexpr (KM > 0) {
#pragma unroll
            for (int s = 0; s < KM; ++s) idx[s] = s < k ? ip[s * inner] : -1;
        }
    }
    __device__ __forceinline__ int index(int s) const {
        if constexpr (KM > 0) return idx[s];
        else return ip[s * inner];
    }
    __device__ __forceinline__ float value(int s) const { return index(s) >= 0 ? vp[s * inner] : -INFINITY; }
    // the class of entry s is none that an entry before it lists
    __device__ __forceinline__ bool first(int s) const {
        bool yes = true;
        for (int q = 0; q < s; ++q) yes &= index(q) != index(s);
        return yes;
    }
};
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// f, or -inf where bit e of w is set
__device__ __forceinline__ float unless(unsigned w, int e, float f) {
    const unsigned m = (unsigned)__builtin_amdgcn_sbfe((int)w, e, 1);
    return __uint_as_float((m & 0xff800000u) | (~m & __float_as_uint(f)));
}
// classes c0 ... in groups of 8: a branch for each class would cost more registers than the classes; past the last class it again
template <typename T, int U>
__device__ __forceinline__ void load_classes(const T* __restrict__ p, int c0, int C, long inner, float* f) {
#pragma unroll
    for (int e0 = 0; e0 < U; e0 += 8)
        if (c0 + e0 < C) {
#pragma unroll
            for (int e = e0; e < e0 + 8; ++e) f[e] = load_elem<T>(p, min(c0 + e, C - 1) * inner);
        }
}
#define LIST_FOR(S) _Pragma("clang loop unroll_count(KM > 0 ? KM : 1)") for (int S = 0; S < (KM > 0 ? KM : list.k); ++S) if (KM == 0 || S < list.k)

template <typename T, int KM>
__global__ void __launch_bounds__(kT) distill_thread_fwd_kernel(const T* __restrict__ z, long ld, int C, long inner, long rows, int k,
                                                                const float* __restrict__ values, const int* __restrict__ indices,
                                                                const float* __restrict__ rest, const unsigned char* __restrict__ mask,
                                                                float temp, float inv_t, float4* __restrict__ stats,
                                                                float* __restrict__ row_loss, double* __restrict__ parts) {
    constexpr int U = kAtOnce;  // classes at a time
    const float c = inv_t * kLog2e;
    double lsum = 0.0, lcount = 0.0;
    for (long row = blockIdx.x * (long)kT + threadIdx.x; row < rows; row += (long)gridDim.x * kT) {
        const long o = (unsigned)row / (unsigned)inner, i = row - o * inner;  // rows fit 31 bits
        const T* p = z + o * ld + i;
        float f[U];
        load_classes<T, U>(p, 0, C, inner, f);
        List<KM> list;
        list.open(values, indices, o, i, inner, k);
        const float r = rest != nullptr ? rest[row] * temp : -INFINITY;
        float vtop = r;
        bool bad = false;
        LIST_FOR(s) {
            const float v = list.value(s);
            vtop = vtop != vtop || v <= vtop ? vtop : v;
            bad |= list.index(s) >= C;
        }
        if (vtop == -INFINITY || (mask != nullptr && mask[row] == 0)) {
            stats[row] = make_float4(0.f, -1.f, 0.f, 0.f);
            if (row_loss != nullptr) row_loss[row] = 0.f;
            continue;
        }
        float zl[KM > 0 ? KM : 1];  // the listed classes' logits: asked for early
        if constexpr (KM > 0) {
#pragma unroll
            for (int s = 0; s < KM; ++s) zl[s] = list.idx[s] >= 0 && list.idx[s] < C ? load_elem<T>(p, list.idx[s] * inner) : -INFINITY;
        }
        LongSum sum;
        for (int c0 = 0; c0 < C; c0 += U) {
            if (c0 > 0) load_classes<T, U>(p, c0, C, inner, f);
            unsigned w = C - c0 < U ? ~0u << (C - c0) : 0u;  // what drops out of the sum: the listed classes, and those past the last
            LIST_FOR(s) {
                const unsigned at = (unsigned)(list.index(s) - c0);
                w |= at < U ? 1u << at : 0u;
            }
            float mu = -INFINITY;
#pragma unroll
            for (int e0 = 0; e0 < U; e0 += 8)
                if (c0 + e0 < C) {
#pragma unroll
                    for (int e = e0; e < e0 + 8; e += 2) {
                        f[e] = unless(w, e, f[e]);
                        f[e + 1] = unless(w, e + 1, f[e + 1]);
                        mu = max3(mu, f[e], f[e + 1]);
                    }
                }
            if (sum.raises(mu, c)) sum.raise(mu, c);
            const float ru = finite_ref(sum.ref);
            float su = 0.f;
#pragma unroll
            for (int e0 = 0; e0 < U; e0 += 8)
                if (c0 + e0 < C) {
#pragma unroll
                    for (int e = e0; e < e0 + 8; ++e) su += exp2_((f[e] - ru) * c);
                }
            sum.add(su);
        }
        const Sum un = {sum.ref, sum.total};
        Sum in = {-INFINITY, 0.f};
        LIST_FOR(s) {
            float zi;
            if constexpr (KM > 0) zi = zl[s];
            else zi = list.index(s) >= 0 && list.index(s) < C ? load_elem<T>(p, list.index(s) * inner) : -INFINITY;
            if (list.first(s)) in = join<false>(in, one(zi), c);
        }
        float4 st = row_stats(un, join<false>(un, in, c));
        if (bad) st.x = st.z = NAN;
        const float ls = log2_sum(st.y), lt = log2_sum(st.w);
        const float lr = (r - vtop) * c;
        float total = exp2_(lr);
        LIST_FOR(s) total += exp2_((list.value(s) - vtop) * c);
        const float L = log2_(total), pr = exp2_(lr - L);
        float loss = 0.f;
        if (pr != 0.f) loss = pr * ((lr - L) - (un.s == 0.f ? -INFINITY : (st.z - st.x) * c + lt - ls));
        LIST_FOR(s) {
            const float lp = (list.value(s) - vtop) * c - L, pi = exp2_(lp);
            const int at = list.index(s);
            float zi;
            if constexpr (KM > 0) zi = zl[s];
            else zi = at >= 0 && at < C ? load_elem<T>(p, at * inner) : 0.f;
            if (pi != 0.f && at >= 0 && at < C) loss += pi * (lp - ((zi - st.x) * c - ls));
        }
        loss = bad ? NAN : temp * temp * kLn2 * loss;
        stats[row] = st;
        if (row_loss != nullptr) row_loss[row] = loss;
        lsum += (double)loss;
        lcount += 1.0;
    }
    leave_part<kT>(lsum, lcount, parts);
}

template <typename T, int KM>
__global__ void __launch_bounds__(kT) distill_thread_bwd_kernel(const T* __restrict__ z, long ld, int C, long inner, long rows, int k,
                                                                const float* __restrict__ values, const int* __restrict__ indices,
                                                                const float* __restrict__ rest, float temp, float inv_t,
                                                                const float4* __restrict__ stats, const float* __restrict__ factor,
                                                                const float* __restrict__ g, int g_rows, T* __restrict__ dz) {
    constexpr int U = 32;
    const float c = inv_t * kLog2e;
    const long row = blockIdx.x * (long)kT + threadIdx.x;
    if (row >= rows) return;
    const long o = (unsigned)row / (unsigned)inner, i = row - o * inner;  // rows fit 31 bits
    const T* p = z + o * ld + i;
    T* d = dz + o * C * inner + i;
    float f[U];
    load_classes<T, U>(p, 0, C, inner, f);  // asked for first: the list and what follows from it come in their shadow
    const float4 st = stats[row];
    // a row that does not count writes its zeros with its neighbours: lines written in two halves cost twice
    const bool counts = row_counts(st);
    List<KM> list;
    list.open(values, indices, o, i, inner, k);
    float zl[KM > 0 ? KM : 1];
    if constexpr (KM > 0) {
#pragma unroll
        for (int s = 0; s < KM; ++s) zl[s] = list.idx[s] >= 0 && list.idx[s] < C ? load_elem<T>(p, list.idx[s] * inner) : 0.f;
    }
    const float r = rest != nullptr ? rest[row] * temp : -INFINITY;
    float vtop = r;
    LIST_FOR(s) {
        const float v = list.value(s);
        vtop = vtop != vtop || v <= vtop ? vtop : v;
    }
    const float wr = exp2_((r - vtop) * c);
    float total = wr;
    LIST_FOR(s) total += exp2_((list.value(s) - vtop) * c);
    const float share_of = part_of(total), q_of = part_of(st.y);
    const float gs = g[g_rows ? row : 0] * (factor != nullptr ? *factor : 1.f) * temp;
    const float outside = gs * (exp2_((st.z - st.x) * c) * (st.w * q_of) - wr * share_of) * part_of(st.w);
    float listed[KM > 0 ? KM : 1];  // the listed classes' gradients
    if constexpr (KM > 0) {
        float pi[KM];
#pragma unroll
        for (int s = 0; s < KM; ++s) pi[s] = s < k ? exp2_((list.value(s) - vtop) * c) * share_of : 0.f;
#pragma unroll
        for (int s = 0; s < KM; ++s) {
            float share = 0.f;
#pragma unroll
            for (int q = 0; q < KM; ++q) share += list.idx[q] == list.idx[s] ? pi[q] : 0.f;
            listed[s] = gs * (exp2_((zl[s] - st.x) * c) * q_of - share);
        }
    }
    for (int c0 = 0; c0 < C; c0 += U) {
        if (c0 > 0) load_classes<T, U>(p, c0, C, inner, f);
#pragma unroll
        for (int e = 0; e < U; ++e)
            if (c0 + e < C) {
                float v = outside * exp2_((f[e] - st.z) * c);
                if constexpr (KM > 0) {
                    LIST_FOR(s) v = list.idx[s] == c0 + e ? listed[s] : v;
                }
                store_elem<T>(d, (c0 + e) * inner, counts ? v : 0.f);
            }
    }
    if (KM == 0 && counts) {
        for (int s = 0; s < k; ++s) {  // the same thread: these stores come after the ones above
            const int at = list.index(s);
            if (at < 0 || at >= C) continue;
            float share = 0.f;
            for (int q = 0; q < k; ++q) share += list.index(q) == at ? exp2_((list.value(q) - vtop) * c) * share_of : 0.f;
            store_elem<T>(d, at * inner, gs * (exp2_((load_elem<T>(p, at * inner) - st.x) * c) * q_of - share));
        }
    }
}

// Rows that one thread takes: maps, whose classes are not adjacent (every map, also one of so few positions that most of the machine
// idles), and short rows where there are very many.  A wave per row costs about 1 ns a row, a thread per row 0.2 us a class however
// few the rows are (selection: 0.2 us up to k = 4, 0.3 (fp32 0.9) up to 16).
// bf16, k = 4, selection / loss by a wave and by a thread: 65536 rows of 64 classes 75 / 61 and 12 / 17 us, 65536 of 128 75 / 65 and
// 21 / 26, 16384 of 64 23 / 20 and 12 / 16, 1024 of 64 7 / 7 and 12 / 16.
bool by_thread(long rows, int classes, long inner, int k, bool select) {
    return inner > 1 || (classes <= 128 && k <= 16 && rows >= classes * (select && k > 4 ? 1024L : 256L));
}

constexpr long kGridThreads = 0xffffffffL;  // of a launch; more rows take several

constexpr int kMaxClasses = 1 << 30;  // an int holds every class a walk steps to, past the last one too

bool layout_ok(long outer, int classes, long inner, long ld) {
    return outer >= 0 && classes > 0 && classes <= kMaxClasses && inner > 0 && (outer <= 1 || ld >= classes * inner) && (inner == 1 || ld == classes * inner) &&
           (outer == 0 || inner <= 0x7fffffffL / outer);
}

// a row's segments: 64 threads x 4 chunks where a row fits, else 256 threads x 8 chunks
int segments(int dtype, int classes) {
    const int vec = msfwsi_vec_of(dtype);
    return classes <= 64 * 4 * vec ? 1 : (classes + 256 * 8 * vec - 1) / (256 * 8 * vec);
}

}  // namespace

#define ST(s) reinterpret_cast<hipStream_t>(s)

extern "C" int msfwsi_top_logits_workspace(int dtype, long outer, int classes, long inner, int k, long* bytes) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && bytes && outer >= 0 && classes > 0 && classes <= kMaxClasses && inner > 0 && k > 0 && k <= kMaxK);
    const int nseg = segments(dtype, classes);
    *bytes = inner > 1 || nseg == 1 ? 0 : outer * nseg * (k + 1L) * 8;
    return MSFWSI_OK;
}

extern "C" int msfwsi_top_logits(int dtype, const void* x, long ld, long outer, int classes, long inner, int k, float inv_t, float* values,
                                 int* indices, float* rest, void* workspace, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && layout_ok(outer, classes, inner, ld) && k > 0 && k <= kMaxK && k <= classes && inv_t > 0.f);
    if (outer == 0) return MSFWSI_OK;
    MSFWSI_CHECK_ARG(x && values && indices && rest);
    if (by_thread(outer, classes, inner, k, true)) {
        const long rows = outer * inner, blocks = (rows + kT - 1) / kT;
#define TOP_THREAD(T, KM, SMALL)                                                                                                  \
    hipLaunchKernelGGL((top_thread_kernel<T, KM, SMALL>), dim3((unsigned)blocks), dim3(kT), 0, ST(stream), (const T*)x, ld, classes, \
                       inner, rows, k, inv_t, values, indices, rest)
#define TOP_THREAD_K(T, SMALL)                   \
    do {                                         \
        if (k <= 4) TOP_THREAD(T, 4, SMALL);     \
        else if (k <= 16) TOP_THREAD(T, 16, SMALL); \
        else TOP_THREAD(T, 64, SMALL);           \
    } while (0)
        if (dtype == MSFWSI_DT_F32) TOP_THREAD_K(float, false);
        else if (classes > 65536) MSFWSI_WITH_T(dtype, TOP_THREAD_K(T, false));
        else if (dtype == MSFWSI_DT_BF16) TOP_THREAD_K(__bf16, true);
        else TOP_THREAD_K(_Float16, true);
        return msfwsi_launch_status();
    }
    const int nseg = segments(dtype, classes);
    const bool narrow = classes <= 64 * 4 * msfwsi_vec_of(dtype);
    if (nseg > 4096) return MSFWSI_EUNSUPPORTED;  // heads of a merge in LDS
    MSFWSI_CHECK_ARG(nseg == 1 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0));
    long* all_keys = (long*)workspace;
    Sum* all_sums = (Sum*)(all_keys + outer * nseg * (long)k);
    const long most = kGridThreads / (kT * (long)nseg);  // rows a launch; a merge takes kT threads a row
    for (long r = 0; r < outer; r += most) {
        const long rows = outer - r < most ? outer - r : most;
        float *v = values + r * k, *re = rest + r;
        int* at = indices + r * k;
        long* keys = all_keys + r * nseg * k;
        Sum* sums = all_sums + r * nseg;
#define TOP_ROWS(NT, NCH, DEEP)                                                                                                           \
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL((top_segment_kernel<T, NT, NCH, DEEP>), dim3((unsigned)(rows * nseg)), dim3(NT), 0, ST(stream), \
                                            (const T*)x + r * ld, ld, classes, nseg, k, inv_t, v, at, re, keys, sums))
        if (narrow && k <= 16) TOP_ROWS(64, 4, false);
        else if (narrow) TOP_ROWS(64, 4, true);
        else TOP_ROWS(256, 8, false);
        int rc = msfwsi_launch_status();
        if (rc != MSFWSI_OK) return rc;
        if (nseg == 1) continue;
        if (nseg * k <= kMergeHeld)
            hipLaunchKernelGGL(top_merge_kernel, dim3((unsigned)rows), dim3(kT), (size_t)nseg * k * 8, ST(stream), keys, sums, nseg, k, inv_t, v, at, re);
        else
            hipLaunchKernelGGL(top_merge_long_kernel, dim3((unsigned)rows), dim3(64), nseg * sizeof(int), ST(stream), keys, sums, nseg, k, inv_t, v, at, re);
        rc = msfwsi_launch_status();
        if (rc != MSFWSI_OK) return rc;
    }
    return MSFWSI_OK;
}

// How many threads take a row of adjacent classes.  One wave (no barriers) for short rows, longer ones too once there are 2048 of them
// (bf16 forward and backward, one wave / 256 threads: 4096 rows of 1000 20 / 31 us, 4096 of 8192 48 / 55, 1024 of 8192 23 / 21,
// fp32 4096 of 16384 179 / 172); 1024 threads where so few long rows leave most of the machine idle (256 / 1024
// threads: 64 rows of 65536 28 / 23 us, 400 rows 41 / 42).
static int row_threads(long rows, int classes) {
    if (classes <= 2048 || (rows >= 2048 && classes <= 8192)) return 64;
    return rows < 256 && classes >= 16384 ? 1024 : 256;
}

extern "C" int msfwsi_distill_fwd(int dtype, const void* z, long ld, long outer, int classes, long inner, int k, const float* values,
                                  const int* indices, const float* rest, const unsigned char* mask, float temperature, int mean, float* stats,
                                  float* row_loss, float* loss, float* factor, double* partials, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && layout_ok(outer, classes, inner, ld) && k > 0 && k <= kMaxK && temperature > 0.f);
    MSFWSI_CHECK_ARG(loss && factor && partials && (reinterpret_cast<uintptr_t>(partials) & 7) == 0);
    long blocks = 0;
    if (outer > 0) {
        MSFWSI_CHECK_ARG(z && values && indices && stats && (reinterpret_cast<uintptr_t>(stats) & 15) == 0);
        const long rows = outer * inner;
        const bool thread = by_thread(rows, classes, inner, k, false);
        const long units = thread ? (rows + kT - 1) / kT : rows;
        const long each = (units + kMaxParts - 1) / kMaxParts;
        blocks = (units + each - 1) / each;
        const float inv_t = 1.f / temperature;
        if (thread) {
#define FWD_THREAD(KM)                                                                                                                   \
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL((distill_thread_fwd_kernel<T, KM>), dim3((unsigned)blocks), dim3(kT), 0, ST(stream),        \
                                            (const T*)z, ld, classes, inner, rows, k, values, indices, rest, mask, temperature, inv_t, \
                                            (float4*)stats, row_loss, partials))
            if (k <= 4) FWD_THREAD(4);
            else if (k <= 16) FWD_THREAD(16);
            else FWD_THREAD(0);
        } else {
#define FWD_ROWS(NT)                                                                                                                 \
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL((distill_fwd_kernel<T, NT>), dim3((unsigned)blocks), dim3(NT), 0, ST(stream),           \
                                            (const T*)z, ld, classes, rows, k, values, indices, rest, mask, temperature, inv_t,     \
                                            (float4*)stats, row_loss, partials))
            const int nt = row_threads(rows, classes);
            if (nt == 64) FWD_ROWS(64);
            else if (nt == 256) FWD_ROWS(256);
            else FWD_ROWS(1024);
        }
        const int rc = msfwsi_launch_status();
        if (rc != MSFWSI_OK) return rc;
    }
    hipLaunchKernelGGL(distill_finish_kernel, dim3(1), dim3(blocks > 1024 ? kFinish : kT), 0, ST(stream), partials, (int)blocks, mean, loss,
                       factor);
    return msfwsi_launch_status();
}

extern "C" int msfwsi_distill_bwd(int dtype, const void* z, long ld, long outer, int classes, long inner, int k, const float* values,
                                  const int* indices, const float* rest, float temperature, const float* stats, const float* factor,
                                  const float* g, int g_rows, void* dz, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && layout_ok(outer, classes, inner, ld) && k > 0 && k <= kMaxK && temperature > 0.f);
    if (outer == 0) return MSFWSI_OK;
    MSFWSI_CHECK_ARG(z && values && indices && stats && (reinterpret_cast<uintptr_t>(stats) & 15) == 0 && g && dz);
    const long rows = outer * inner;
    const float inv_t = 1.f / temperature;
    if (by_thread(rows, classes, inner, k, false)) {
#define BWD_THREAD(KM)                                                                                                                      \
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL((distill_thread_bwd_kernel<T, KM>), dim3((unsigned)((rows + kT - 1) / kT)), dim3(kT), 0,       \
                                            ST(stream), (const T*)z, ld, classes, inner, rows, k, values, indices, rest, temperature,     \
                                            inv_t, (const float4*)stats, factor, g, g_rows, (T*)dz))
        if (k <= 4) BWD_THREAD(4);
        else if (k <= 16) BWD_THREAD(16);
        else BWD_THREAD(0);
        return msfwsi_launch_status();
    }
    const int nt = row_threads(rows, classes);
    const long most = kGridThreads / nt;
    for (long r = 0; r < rows; r += most) {
        const long n = rows - r < most ? rows - r : most;
#define BWD_ROWS(NT)                                                                                                                          \
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL((distill_bwd_kernel<T, NT>), dim3((unsigned)n), dim3(NT), 0, ST(stream), (const T*)z + r * ld, ld, \
                                            classes, n, k, values + r * k, indices + r * k, rest != nullptr ? rest + r : nullptr, temperature, \
                                            inv_t, (const float4*)stats + r, factor, g + (g_rows ? r : 0), g_rows, (T*)dz + r * classes))
        if (nt == 64) BWD_ROWS(64);
        else if (nt == 256) BWD_ROWS(256);
        else BWD_ROWS(1024);
        const int rc = msfwsi_launch_status();
        if (rc != MSFWSI_OK) return rc;
    }
    return MSFWSI_OK;
}
