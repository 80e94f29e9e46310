// Microscaled 4-bit storage (blocks of 32 elements under one 8-bit power-of-two scale) and its products: quantisation,
// widening, y = x W^T on the 4-bit matrix instructions, and the input gradient dx = dy W of a frozen W.
//
// Format.  A row of `cols` elements is cut into groups of 256 (the last one filled up with zeros): 128 bytes of codes --
// element 2i in the low four bits of byte i, element 2i + 1 in the high four -- and 8 scale bytes, one per 32 elements.  Groups
// are the OUTER dimension, codes [G][rows][128] and scales [G][rows][8]: the rows of one group are contiguous, so a tile of
// rows x 256 elements is ONE run of memory for every reader.
//   code    sign bit 3, then {0, .5, 1, 1.5, 2, 3, 4, 6}
//   scale   E stands for 2^(E - 127); E = 255 makes the whole block NaN
// A block's scale is E = max(exponent field of its largest magnitude - 2, 0): the largest magnitude falls into [4, 8) of the
// scaled range; elements round to nearest (ties to the even code) and saturate at 6.  A block with an infinity or a NaN gets
// E = 255, so that it cannot pass unnoticed through a product.
#include "common.h"
#include "../../include/msfwsi_hip.h"

namespace {

constexpr int kGroup = 256;             // elements of a row that are stored together
constexpr int kGroupBytes = kGroup / 2; // their codes
constexpr int kT = 256;

typedef __attribute__((ext_vector_type(8))) int i32x8;

// 2^(E - 127) as fp32, exact (E = 0 is the subnormal 2^-127; E = 255 a NaN)
__device__ __forceinline__ float scale_value(unsigned E) {
    return __uint_as_float(E == 0 ? 0x00400000u : E == 255u ? 0x7fc00000u : E << 23);
}

__device__ __forceinline__ float code_value(unsigned c) {
    const unsigned m = c & 7u;
    const float v = m < 4 ? 0.5f * (float)m : m == 4 ? 2.f : m == 5 ? 3.f : m == 6 ? 4.f : 6.f;
    return (c & 8u) ? -v : v;
}

template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, long left, float* f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < left ? load_elem<T>(p, e) : 0.f;
}

// One half-wave (32 lanes x 8 elements) per group of a row; a block of 32 elements is 4 lanes.  The conversion's own scale
// operand stays 1: the elements are multiplied by 2^(127 - E) first, which is exact.
template <typename T>
__global__ void __launch_bounds__(kT) mx4_quantize_kernel(const T* __restrict__ x, long ld, long rows, long cols,
                                                          unsigned* __restrict__ codes, unsigned* __restrict__ scales) {
    const int l = threadIdx.x & 31;
    const long r = blockIdx.x * (long)(kT / 32) + (threadIdx.x >> 5), g = blockIdx.y;
    if (r >= rows) return;  // whole half-waves leave; the shuffles below stay inside a half
    const long c = g * kGroup + l * 8;
    float f[8];
    load8<T>(x + r * ld + c, cols - c, f);
    unsigned big = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) big = max(big, __float_as_uint(f[e]) & 0x7fffffffu);  // orders like the magnitudes, NaN on top
    big = max(big, (unsigned)__shfl_xor((int)big, 1, 64));
    big = max(big, (unsigned)__shfl_xor((int)big, 2, 64));
    const unsigned field = big >> 23;
    const unsigned E = field == 255u ? 255u : field > 2u ? field - 2u : 0u;
    const float up = __uint_as_float((254u - (E == 255u ? 127u : E)) << 23);  // 2^(127 - E)
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0] * up, f[1] * up, 1.f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2] * up, f[3] * up, 1.f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4] * up, f[5] * up, 1.f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6] * up, f[7] * up, 1.f, 3);
    if (E == 255u) w = 0;
    codes[(g * rows + r) * 32 + l] = w;
    unsigned word = 0;  // lane 0 / 1 collects the scale bytes of blocks 0-3 / 4-7
#pragma unroll
    for (int j = 0; j < 4; ++j) word |= (unsigned)__shfl((int)E, (threadIdx.x & 32) + (l & 1) * 16 + j * 4, 64) << (8 * j);
    if (l < 2) scales[(g * rows + r) * 2 + l] = word;
}

template <typename T>
__global__ void __launch_bounds__(kT) mx4_dequantize_kernel(const unsigned* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                            long rows, long cols, T* __restrict__ y) {
    const int l = threadIdx.x & 31;
    const long r = blockIdx.x * (long)(kT / 32) + (threadIdx.x >> 5), g = blockIdx.y;
    if (r >= rows) return;
    const long c = g * kGroup + l * 8;
    const unsigned w = codes[(g * rows + r) * 32 + l];
    const float s = scale_value(scales[(g * rows + r) * 8 + (l >> 2)]);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (c + e < cols) store_elem<T>(y, r * cols + c + e, code_value(w >> (4 * e)) * s);
}

// y = a b^T (+ bias): 32 x 32 outputs per workgroup, the groups dealt over its four waves and joined in LDS.
// A 32x32x64 step takes 32 elements of row (lane & 31) from each lane; which 32 is free as long as both operands agree, so
// half h of the wave takes block 4h + s in step s: its four scales are then one aligned dword and step s reads byte s of it.
template <typename T>
__global__ void __launch_bounds__(kT) mx4_gemm_kernel(const unsigned char* __restrict__ a, const unsigned char* __restrict__ as, long M,
                                                      const unsigned char* __restrict__ b, const unsigned char* __restrict__ bs, long N,
                                                      int G, const float* __restrict__ bias, T* __restrict__ y, unsigned nt) {
    __shared__ float part[4][32 * 33];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
    const long m0 = (long)(blockIdx.x / nt) * 32, n0 = (long)(blockIdx.x % nt) * 32;
    const long m = min(m0 + (lane & 31), M - 1), n = min(n0 + (lane & 31), N - 1);
    f32x16 acc = {0.f};
    for (int g = w; g < G; g += 4) {
        const long ra = g * M + m, rb = g * N + n;
        const int sa = *reinterpret_cast<const int*>(as + ra * 8 + h * 4), sb = *reinterpret_cast<const int*>(bs + rb * 8 + h * 4);
        int4 fa[4], fb[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            fa[s] = *reinterpret_cast<const int4*>(a + ra * kGroupBytes + (4 * h + s) * 16);
            fb[s] = *reinterpret_cast<const int4*>(b + rb * kGroupBytes + (4 * h + s) * 16);
        }
#define MX4_STEP(S)                                                                                                          \
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4((i32x8){fa[S].x, fa[S].y, fa[S].z, fa[S].w, 0, 0, 0, 0},           \
                                                          (i32x8){fb[S].x, fb[S].y, fb[S].z, fb[S].w, 0, 0, 0, 0}, acc, 4, 4, \
                                                          S, sa, S, sb)
        MX4_STEP(0);
        MX4_STEP(1);
        MX4_STEP(2);
        MX4_STEP(3);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) part[w][((i & 3) + 8 * (i >> 2) + 4 * h) * 33 + (lane & 31)] = acc[i];
    __syncthreads();
    for (int i = threadIdx.x; i < 1024; i += kT) {
        const int r = i >> 5, c = i & 31;
        if (m0 + r >= M || n0 + c >= N) continue;
        float v = (part[0][r * 33 + c] + part[1][r * 33 + c]) + (part[2][r * 33 + c] + part[3][r * 33 + c]);
        if (bias != nullptr) v += bias[n0 + c];
        store_elem<T>(y, (m0 + r) * N + n0 + c, v);
    }
}

// dx = dy W: 32 rows x 32 columns (one scale block) per workgroup, the rows of W dealt over its four waves.  W widens to
// bf16 exactly (two mantissa bits); dy in fp16 / fp32 is cut into 2 / 3 bf16 parts that add up to it exactly, so every
// product is exact and the sums are fp32.
template <typename T, typename TO>
__global__ void __launch_bounds__(kT) mx4_dgrad_kernel(const T* __restrict__ dy, long ld, long M, const unsigned char* __restrict__ codes,
                                                       const unsigned char* __restrict__ scales, long N, long cols, TO* __restrict__ dx,
                                                       unsigned kt) {
    constexpr int PARTS = sizeof(T) == 4 ? 3 : __is_same(T, _Float16) ? 2 : 1;
    __shared__ float part[4][32 * 33];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5, l = lane & 31;
    const long m0 = (long)(blockIdx.x / kt) * 32, k0 = (long)(blockIdx.x % kt) * 32;
    const long m = min(m0 + l, M - 1), g = k0 / kGroup;
    const int kb = (int)(k0 % kGroup) / 32;
    f32x16 acc = {0.f};
    for (long n0 = w * 16; n0 < N; n0 += 64) {
        bf16x8 fa[PARTS], fb;
        float v[8];
        load8<T>(dy + m * ld + n0 + h * 8, N - n0 - h * 8, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float left = v[e];
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                const float top = p + 1 < PARTS ? __uint_as_float(__float_as_uint(left) & 0xffff0000u) : left;
                fa[p][e] = (__bf16)top;
                left = top == left ? 0.f : left - top;
            }
            const long n = n0 + h * 8 + e;
            float c = 0.f;
            if (n < N)
                c = code_value(codes[(g * N + n) * kGroupBytes + kb * 16 + (l >> 1)] >> (4 * (l & 1))) * scale_value(scales[(g * N + n) * 8 + kb]);
            fb[e] = (__bf16)c;
        }
#pragma unroll
        for (int p = 0; p < PARTS; ++p) mma32<__bf16>(acc, fa[p], fb);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) part[w][((i & 3) + 8 * (i >> 2) + 4 * h) * 33 + l] = acc[i];
    __syncthreads();
    for (int i = threadIdx.x; i < 1024; i += kT) {
        const int r = i >> 5, c = i & 31;
        if (m0 + r >= M || k0 + c >= cols) continue;
        store_elem<TO>(dx, (m0 + r) * cols + k0 + c, (part[0][r * 33 + c] + part[1][r * 33 + c]) + (part[2][r * 33 + c] + part[3][r * 33 + c]));
    }
}

long groups_of(long cols) { return (cols + kGroup - 1) / kGroup; }
bool grid_ok(long blocks) { return blocks > 0 && blocks <= 0xffffffL; }  // a grid holds fewer than 2^32 threads

}  // namespace

#define ST(s) reinterpret_cast<hipStream_t>(s)

extern "C" int msfwsi_mx4_quantize(int dtype, const void* x, long ld, long rows, long cols, void* codes, void* scales, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && rows >= 0 && cols > 0 && (rows <= 1 || ld >= cols));
    if (rows == 0) return MSFWSI_OK;
    const long G = groups_of(cols);
    MSFWSI_CHECK_ARG(x && codes && scales && G <= 65535 && grid_ok((rows + 7) / 8));
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL(mx4_quantize_kernel<T>, dim3((unsigned)((rows + 7) / 8), (unsigned)G), dim3(kT), 0, ST(stream),
                                            (const T*)x, ld, rows, cols, (unsigned*)codes, (unsigned*)scales));
    return msfwsi_launch_status();
}

extern "C" int msfwsi_mx4_dequantize(int dtype, const void* codes, const void* scales, long rows, long cols, void* y, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && rows >= 0 && cols > 0);
    if (rows == 0) return MSFWSI_OK;
    const long G = groups_of(cols);
    MSFWSI_CHECK_ARG(y && codes && scales && G <= 65535 && grid_ok((rows + 7) / 8));
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL(mx4_dequantize_kernel<T>, dim3((unsigned)((rows + 7) / 8), (unsigned)G), dim3(kT), 0, ST(stream),
                                            (const unsigned*)codes, (const unsigned char*)scales, rows, cols, (T*)y));
    return msfwsi_launch_status();
}

extern "C" int msfwsi_mx4_gemm(int dtype, const void* a_codes, const void* a_scales, long M, const void* b_codes, const void* b_scales,
                               long N, long cols, const float* bias, void* y, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && M >= 0 && N > 0 && cols > 0);
    if (M == 0) return MSFWSI_OK;
    const long mt = (M + 31) / 32, nt = (N + 31) / 32, G = groups_of(cols);
    MSFWSI_CHECK_ARG(a_codes && a_scales && b_codes && b_scales && y && G <= 0x7fffffffL && nt <= 0x7fffffffL && mt <= 0x7fffffffL && grid_ok(mt * nt));
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL(mx4_gemm_kernel<T>, dim3((unsigned)(mt * nt)), dim3(kT), 0, ST(stream),
                                            (const unsigned char*)a_codes, (const unsigned char*)a_scales, M, (const unsigned char*)b_codes,
                                            (const unsigned char*)b_scales, N, (int)G, bias, (T*)y, (unsigned)nt));
    return msfwsi_launch_status();
}

extern "C" int msfwsi_mx4_dgrad(int dy_dtype, const void* dy, long ld, long M, const void* codes, const void* scales, long N, long cols,
                                int dx_dtype, void* dx, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dy_dtype) && msfwsi_dtype_ok(dx_dtype) && M >= 0 && N > 0 && cols > 0 && (M <= 1 || ld >= N));
    if (M == 0) return MSFWSI_OK;
    const long mt = (M + 31) / 32, kt = (cols + 31) / 32;
    MSFWSI_CHECK_ARG(dy && codes && scales && dx && kt <= 0x7fffffffL && mt <= 0x7fffffffL && grid_ok(mt * kt));
#define MX4_DGRAD(TO)                                                                                                              \
    MSFWSI_WITH_T(dy_dtype, hipLaunchKernelGGL((mx4_dgrad_kernel<T, TO>), dim3((unsigned)(mt * kt)), dim3(kT), 0, ST(stream),     \
                                               (const T*)dy, ld, M, (const unsigned char*)codes, (const unsigned char*)scales, N, \
                                               cols, (TO*)dx, (unsigned)kt))
    if (dx_dtype == MSFWSI_DT_BF16) {
        MX4_DGRAD(__bf16);
    } else if (dx_dtype == MSFWSI_DT_F16) {
        MX4_DGRAD(_Float16);
    } else {
        MX4_DGRAD(float);
    }
    return msfwsi_launch_status();
}
