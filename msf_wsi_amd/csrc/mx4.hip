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

#include <type_traits>

namespace {

constexpr int kGroup = 256;             // elements of a row that are stored together
constexpr int kGroupBytes = kGroup / 2; // their codes
constexpr int kT = 256;

typedef __attribute__((ext_vector_type(8))) int i32x8;

// 2^(E - 127) as fp32, exact (E = 0 is the subnormal 2^-127; E = 255 a NaN)
__device__ __forceinline__ float scale_value(unsigned E) {
    return __uint_as_float(E == 0 ? 0x00400000u : E == 255u ? 0x7fc00000u : E << 23);
}

// 8 elements of a row at any alignment, zeros past its end; `left` = elements from here to the end
struct __attribute__((packed, aligned(2))) Unaligned16 {
    unsigned x, y, z, w;
};
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, long left, float* f) {
    if (left >= 8) {
#pragma unroll
        for (int i = 0; i < 8 / ElemTraits<T>::VEC; ++i) {
            const Unaligned16 u = reinterpret_cast<const Unaligned16*>(p)[i];
            unpack16<T>(make_uint4(u.x, u.y, u.z, u.w), f + i * ElemTraits<T>::VEC);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < left ? load_elem<T>(p, e) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, long left, const float* f) {
    if (left >= 8) {
#pragma unroll
        for (int i = 0; i < 8 / ElemTraits<T>::VEC; ++i) {
            const uint4 v = pack16<T>(f + i * ElemTraits<T>::VEC);
            reinterpret_cast<Unaligned16*>(p)[i] = {v.x, v.y, v.z, v.w};
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < left) store_elem<T>(p, e, f[e]);
}

// 8 elements of a block whose other 24 are in the neighbouring lanes (4 lanes from a multiple of 4): their codes, the block's E.
// The conversion's own scale operand stays 1: the elements are multiplied by 2^(127 - E) first, which is exact.
__device__ __forceinline__ unsigned quantize8(const float* f, unsigned& E) {
    unsigned big = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) big = max(big, __float_as_uint(f[e]) & 0x7fffffffu);  // orders like the magnitudes, NaN on top
    big = max(big, (unsigned)__shfl_xor((int)big, 1, 64));
    big = max(big, (unsigned)__shfl_xor((int)big, 2, 64));
    const unsigned field = big >> 23;
    E = field == 255u ? 255u : field > 2u ? field - 2u : 0u;
    const float up = __uint_as_float((254u - (E == 255u ? 127u : E)) << 23);  // 2^(127 - E)
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0] * up, f[1] * up, 1.f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2] * up, f[3] * up, 1.f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4] * up, f[5] * up, 1.f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6] * up, f[7] * up, 1.f, 3);
    return E == 255u ? 0u : w;
}

// One half-wave (32 lanes x 8 elements) per group of a row, UG groups one after the other with their loads in flight together.
// Bound by memory: 18432 x 18432 fp32 quantised in 346 us (4.5 TB/s read and written), widened to fp32 in 309 us (5.0 TB/s).
constexpr int UG = 4;
template <typename T>
__global__ void __launch_bounds__(kT) mx4_quantize_kernel(const T* __restrict__ x, long ld, long rows, long cols, int G,
                                                          unsigned* __restrict__ codes, unsigned* __restrict__ scales) {
    const int l = threadIdx.x & 31, g0 = blockIdx.y * UG;
    const long r = blockIdx.x * (long)(kT / 32) + (threadIdx.x >> 5);
    if (r >= rows) return;  // whole half-waves leave; the shuffles below stay inside a half
    float f[UG][8];
#pragma unroll
    for (int u = 0; u < UG; ++u) {
        const long c = (g0 + u) * (long)kGroup + l * 8;
        load8<T>(x + r * ld + c, cols - c, f[u]);  // nothing is read of a group past the last
    }
#pragma unroll
    for (int u = 0; u < UG; ++u) {
        if (g0 + u >= G) return;
        const long at = (long)(g0 + u) * rows + r;
        unsigned E;
        codes[at * 32 + l] = quantize8(f[u], E);
        unsigned word = 0;  // lane 0 / 1 collects the scale bytes of blocks 0-3 / 4-7
#pragma unroll
        for (int j = 0; j < 4; ++j) word |= (unsigned)__shfl((int)E, (threadIdx.x & 32) + (l & 1) * 16 + j * 4, 64) << (8 * j);
        if (l < 2) scales[at * 2 + l] = word;
    }
}

typedef __attribute__((ext_vector_type(2))) float f32x2;
template <typename T>
__global__ void __launch_bounds__(kT) mx4_dequantize_kernel(const unsigned* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                            long rows, long cols, int G, T* __restrict__ y) {
    const int l = threadIdx.x & 31, g0 = blockIdx.y * UG;
    const long r = blockIdx.x * (long)(kT / 32) + (threadIdx.x >> 5);
    if (r >= rows) return;
    unsigned w[UG], E[UG];
#pragma unroll
    for (int u = 0; u < UG; ++u) {
        const long at = (long)min(g0 + u, G - 1) * rows + r;
        w[u] = codes[at * 32 + l];
        E[u] = scales[at * 8 + (l >> 2)];
    }
#pragma unroll
    for (int u = 0; u < UG; ++u) {
        if (g0 + u >= G) return;
        const long c = (g0 + u) * (long)kGroup + l * 8;
        const float s = scale_value(E[u]);
        float f[8];
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.f, 1);
        const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.f, 3);
        f[0] = a.x * s, f[1] = a.y * s, f[2] = b.x * s, f[3] = b.y * s, f[4] = d.x * s, f[5] = d.y * s, f[6] = e.x * s, f[7] = e.y * s;
        store8<T>(y + r * cols + c, cols - c, f);
    }
}
// fp32 results are 32 bytes a lane: here a lane takes four elements of either half of the group, so that a store covers whole lines
__global__ void __launch_bounds__(kT) mx4_dequantize32_kernel(const unsigned short* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                              long rows, long cols, int G, float* __restrict__ y) {
    const int l = threadIdx.x & 31, g0 = blockIdx.y * UG;
    const long r = blockIdx.x * (long)(kT / 32) + (threadIdx.x >> 5);
    if (r >= rows) return;
    unsigned w[2 * UG], E[2 * UG];
#pragma unroll
    for (int u = 0; u < 2 * UG; ++u) {
        const long at = (long)min(g0 + u / 2, G - 1) * rows + r;
        w[u] = codes[at * 64 + (u & 1) * 32 + l];
        E[u] = scales[at * 8 + (u & 1) * 4 + (l >> 3)];
    }
#pragma unroll
    for (int u = 0; u < 2 * UG; ++u) {
        const long c = (g0 + u / 2) * (long)kGroup + (u & 1) * 128 + l * 4;
        const float s = scale_value(E[u]);
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.f, 1);
        const float f[4] = {a.x * s, a.y * s, b.x * s, b.y * s};
        float* p = y + r * cols + c;
        if (c + 4 <= cols) {
            *reinterpret_cast<Unaligned16*>(p) = {__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < cols) p[e] = f[e];
        }
    }
}

// One 32x32x64 step takes 32 elements of row (lane & 31) of either operand from each lane.  Which 32 is free as long as both
// operands agree: half h of the wave takes block 4h + S of a group in step S, so its four scales are one aligned dword, of which
// step S reads byte S.
template <int S>
__device__ __forceinline__ void mx4_step(f32x16& acc, const int4& a, int sa, const int4& b, int sb) {
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4((i32x8){a.x, a.y, a.z, a.w, 0, 0, 0, 0}, (i32x8){b.x, b.y, b.z, b.w, 0, 0, 0, 0},
                                                          acc, 4, 4, S, sa, S, sb);
}

// Few rows (up to 16 FA): 16 columns per workgroup straight from memory, the groups dealt over its NW waves and joined in LDS.
// Bound by reading b once; nothing is shared between workgroups, so nothing is staged, and the next group's loads are on their
// way while one is multiplied.  16 columns, because a CU's share is a whole number of workgroups: 576 of 32 columns on 256 CUs
// (18432 rows of b) took 51 us, 1152 of 16 took 40.
// A 16x16x128 step takes 32 elements from each lane; quarter q of the wave takes blocks 2q, 2q + 1 of a group in its two steps.
// ROW: a single row of up to kRowGroups groups, which comes as it is (TX) and is quantised by every workgroup for itself, so that one
// launch does it all; the codes wait in LDS.  (One group after the other, with its loads waited for, this took 13 us.)
constexpr int kRowGroups = 128;
template <int S>
__device__ __forceinline__ void mx4_step16(f32x4& acc, const int4& a, int sa, const int4& b, int sb) {
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4((i32x8){a.x, a.y, a.z, a.w, 0, 0, 0, 0}, (i32x8){b.x, b.y, b.z, b.w, 0, 0, 0, 0},
                                                           acc, 4, 4, S, sa, S, sb);
}
template <typename T, typename TX, bool ROW, int FA, int NW>
__global__ void __launch_bounds__(NW * 64) mx4_gemm_kernel(const void* __restrict__ a, const unsigned char* __restrict__ as, long M, long cols,
                                                           const unsigned char* __restrict__ b, const unsigned char* __restrict__ bs, long N,
                                                           int G, const float* __restrict__ bias, T* __restrict__ y) {
    __shared__ float part[NW][ROW ? 16 : FA * 16 * 17];
    __shared__ __attribute__((aligned(16))) unsigned char own[ROW ? kRowGroups * (kGroupBytes + 16) : 16];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, l = lane & 15;
    const long n0 = blockIdx.x * 16L, n = min(n0 + l, N - 1);
    struct Operands {
        int4 a[FA][2], b[2];
        int sa[FA], sb;
    } first, second;
    auto load = [&](int g, Operands& o) {
        if constexpr (!ROW) {
#pragma unroll
            for (int i = 0; i < FA; ++i) {
                const long ra = g * M + min(i * 16L + l, M - 1);
                o.sa[i] = *reinterpret_cast<const unsigned short*>(as + ra * 8 + q * 2);
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    o.a[i][s] = *reinterpret_cast<const int4*>(reinterpret_cast<const unsigned char*>(a) + ra * kGroupBytes + (2 * q + s) * 16);
            }
        }
        const long rb = g * N + n;
        o.sb = *reinterpret_cast<const unsigned short*>(bs + rb * 8 + q * 2);
#pragma unroll
        for (int s = 0; s < 2; ++s) o.b[s] = *reinterpret_cast<const int4*>(b + rb * kGroupBytes + (2 * q + s) * 16);
    };
    f32x4 acc[FA];
#pragma unroll
    for (int i = 0; i < FA; ++i) acc[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](int g, Operands& o) {
        if constexpr (ROW) {
            const unsigned char* x = own + g * (kGroupBytes + 16);
            o.sa[0] = *reinterpret_cast<const unsigned short*>(x + kGroupBytes + q * 2);
#pragma unroll
            for (int s = 0; s < 2; ++s) o.a[0][s] = *reinterpret_cast<const int4*>(x + (2 * q + s) * 16);
        }
#pragma unroll
        for (int i = 0; i < FA; ++i) {
            mx4_step16<0>(acc[i], o.a[i][0], o.sa[i], o.b[0], o.sb);
            mx4_step16<1>(acc[i], o.a[i][1], o.sa[i], o.b[1], o.sb);
        }
    };
    load(min(w, G - 1), first);
    if constexpr (ROW) {  // half a wave per group, 8 elements a lane (mx4_quantize_kernel), all loads of five groups in flight
        constexpr int H = 2 * NW, U = 5;
        const int hl = threadIdx.x & 31;
        for (int g = threadIdx.x >> 5; g < G; g += H * U) {
            float f[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long c = (g + u * H) * (long)kGroup + hl * 8;
                load8<TX>(reinterpret_cast<const TX*>(a) + c, cols - c, f[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (g + u * H >= G) break;
                unsigned E;
                const unsigned code = quantize8(f[u], E);
                unsigned char* x = own + (g + u * H) * (kGroupBytes + 16);
                *reinterpret_cast<unsigned*>(x + hl * 4) = code;
                if ((hl & 3) == 0) x[kGroupBytes + (hl >> 2)] = (unsigned char)E;
            }
        }
        __syncthreads();
    }
    int g = w;
    for (; g + NW < G; g += 2 * NW) {  // two sets of registers in turn: a copy from one to the other would wait for its loads
        load(g + NW, second);
        __builtin_amdgcn_sched_barrier(0);  // and neither set's loads move behind the other's products
        multiply(g, first);
        load(min(g + 2 * NW, G - 1), first);
        __builtin_amdgcn_sched_barrier(0);
        multiply(g + NW, second);
    }
    if (g < G) multiply(g, first);
    if constexpr (ROW) {  // all 16 rows of the operand are this one
        if (lane < 16) part[w][lane] = acc[0][0];
    } else {
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[w][(i * 16 + q * 4 + e) * 17 + l] = acc[i][e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < (ROW ? 16 : FA * 256); i += NW * 64) {
        const int r = i >> 4, c = i & 15;
        if (r >= M || n0 + c >= N) continue;
        float v = 0.f;
#pragma unroll
        for (int p = 0; p < NW; ++p) v += part[p][r * 17 + c];
        if (bias != nullptr) v += bias[n0 + c];
        store_elem<T>(y, r * N + n0 + c, v);
    }
}

// 16 (4) bytes per lane global -> LDS, lane l to base + 16 l (4 l): lds_dma16_buf of common.h, whose rules for waits hold here
// too, with a constant part of the byte offset added inside -- as an operand of its own it took a register per request
template <int BYTES>
__device__ __forceinline__ void lds_dma(__amdgpu_buffer_rsrc_t rsrc, void* lds_wave_base, int voff, int more) {
    const unsigned lds = (unsigned)(__UINTPTR_TYPE__)(__attribute__((address_space(3))) char*)lds_wave_base;
    int at;
    if constexpr (BYTES == 16)
        asm volatile("s_mov_b32 m0, %1\n\tv_add_u32 %0, %3, %2\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %4, 0 offen lds"
                     : "=&v"(at)
                     : "s"(lds), "v"(voff), "s"(more), "s"(rsrc)
                     : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %1\n\tv_add_u32 %0, %3, %2\n\ts_nop 3\n\tbuffer_load_dword %0, %4, 0 offen lds"
                     : "=&v"(at)
                     : "s"(lds), "v"(voff), "s"(more), "s"(rsrc)
                     : "memory", "m0");
}
// the address and the size are the same in all lanes, which hipcc does not see through a select
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const unsigned char* p, long bytes) {
    const unsigned long u = reinterpret_cast<unsigned long>(p);
    const unsigned lo = __builtin_amdgcn_readfirstlane((int)u), hi = __builtin_amdgcn_readfirstlane((int)(u >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((unsigned long)hi << 32) | lo), 0,
                                             __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}
// everything this wave has asked for has arrived, and it is done reading the stage it leaves; then all waves
__device__ __forceinline__ void stage_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Two adjacent results of one row, at any alignment; the second only where the row has it.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Two {
    T a, b;
};
template <typename T>
__device__ __forceinline__ void store_two(T* p, unsigned at, float a, float b, bool both) {
    if (both) *reinterpret_cast<Two<T>*>(p + at) = {(T)a, (T)b};
    else p[at] = (T)a;
}

// Tiles go to the XCDs in contiguous runs (xcd_remap), inside a run down columns of 8 row tiles: a run then shares few row and
// column tiles in its L2.
__device__ __forceinline__ void tile_of(unsigned id, unsigned mt, unsigned nt, unsigned& m, unsigned& n) {
    const unsigned wide = 8 * nt, first = id / wide * 8, deep = min(mt - first, 8u), in = id % wide;
    m = first + in % deep;
    n = in / deep;
}

struct GemmArgs {
    const unsigned char *a, *as, *b, *bs;
    long M, N;
    int G, per_split;
    const float* bias;
    void* y;
    float* sums;  // not NULL: the groups of a tile are dealt over several workgroups, which leave fp32 sums [split][M][N] for a join
    unsigned mt, nt;
};

// Many rows: TM x TN outputs per workgroup of WM x WN waves, one group of 256 elements (128 bytes of every row) per stage, two
// stages in LDS filled by DMA.  A row's eight 16-byte chunks lie at (chunk ^ (row / 2 & 7)): the sixteen rows that a read takes
// at a time then fall on all 64 banks.  The columns of a wave's 64 are dealt to its two fragments in turn (2 l + j: b's rows lie in
// LDS in that order), so that a lane ends up with neighbours of a row and a wave writes whole 128-byte lines.
// 8192 x 9216 x 9216: 376 us, 3.7 PFLOP/s (4.5 rounds of tiles); 8192 x 8192 x 8192: 290 us, 3.8 PFLOP/s (registers alone reach 6.5
// at this card's power).  Requests and
// products share the CU's LDS and issue slots; a four-stage ring of half groups (64-byte lines: 0.8 of the rate), fragments
// read a step ahead by hand, a workgroup that runs through its tiles, and four waves of 128 x 128 were all 2 - 20 % slower.
template <typename T, int TM, int TN, int WM, int WN>
__global__ void __launch_bounds__(WM* WN * 64) mx4_tile_kernel(const GemmArgs p) {
    constexpr int NW = WM * WN, FM = TM / WM / 32, FN = 2;
    static_assert(TN / WN == 64, "a wave has 64 columns");
    constexpr int kStage = (TM + TN) * (kGroupBytes + 8);
    constexpr int PA = TM / 8 / NW, PB = TN / 8 / NW, PSA = TM / 32 / NW, PSB = TN / 32 / NW, PIECES = PA + PB + PSA + PSB;
    __shared__ __attribute__((aligned(1024))) char smem[2 * kStage];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, l = lane & 31;
    const int swz = ((lane & 7) ^ ((w & 1) * 4 + (lane >> 4))) << 4;  // of row (lane >> 3) of any 1 KB piece this wave brings
    const int chunk_a = (lane >> 3) * kGroupBytes + swz, chunk_b = (lane >> 3) * 2 * kGroupBytes + swz;

    const unsigned it = xcd_remap(blockIdx.x, gridDim.x), tiles = p.mt * p.nt, split = it / tiles;
    unsigned tm, tn;
    tile_of(it % tiles, p.mt, p.nt, tm, tn);
    const long m0 = (long)tm * TM, n0 = (long)tn * TN;
    const int mrows = (int)min((long)TM, p.M - m0), nrows = (int)min((long)TN, p.N - n0);
    const int g0 = (int)split * p.per_split, g1 = min(p.G, g0 + p.per_split);
    __amdgpu_buffer_rsrc_t ra, rb, rsa, rsb;
    auto aim = [&](int g) {
        ra = buffer_of(p.a + (g * p.M + m0) * kGroupBytes, mrows * kGroupBytes);
        rb = buffer_of(p.b + (g * p.N + n0) * kGroupBytes, nrows * kGroupBytes);
        rsa = buffer_of(p.as + (g * p.M + m0) * 8, mrows * 8);
        rsb = buffer_of(p.bs + (g * p.N + n0) * 8, nrows * 8);
    };
    auto piece = [&](char* st, int i) {
        char* sc = st + (TM + TN) * kGroupBytes;
        const int j = i < PA ? i : i < PA + PB ? i - PA : i < PA + PB + PSA ? i - PA - PB : i - PA - PB - PSA, q = j * NW + w;
        if (i < PA) lds_dma<16>(ra, st + q * 1024, chunk_a, q * 1024);
        else if (i < PA + PB) lds_dma<16>(rb, st + TM * kGroupBytes + q * 1024, chunk_b, ((q >> 3) * 64 + (q & 3) * 16 + ((q >> 2) & 1)) * kGroupBytes);
        else if (i < PA + PB + PSA) lds_dma<4>(rsa, sc + q * 256, lane * 4, q * 256);
        else lds_dma<4>(rsb, sc + TM * 8 + q * 256, lane * 4, q * 256);
    };
    f32x16 acc[FM][FN];
    const int wm = w / WN, wn = w % WN;
    const int arow = wm * (TM / WM) + l, brow = wn * 64 + l;
    auto compute = [&](const char* st) {
        const char* sc = st + (TM + TN) * kGroupBytes + h * 4;
        int sa[FM], sb[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) sa[i] = *reinterpret_cast<const int*>(sc + (arow + i * 32) * 8);
#pragma unroll
        for (int j = 0; j < FN; ++j) sb[j] = *reinterpret_cast<const int*>(sc + (TM + wn * 64 + 2 * l + j) * 8);
        auto step = [&](auto s_) {
            constexpr int S = decltype(s_)::value;
            const int at = ((4 * h + S) ^ ((l >> 1) & 7)) << 4;
            int4 fa[FM], fb[FN];
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[i] = *reinterpret_cast<const int4*>(st + (arow + i * 32) * kGroupBytes + at);
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[j] = *reinterpret_cast<const int4*>(st + (TM + brow + j * 32) * kGroupBytes + at);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) mx4_step<S>(acc[i][j], fa[i], sa[i], fb[j], sb[j]);
        };
        step(std::integral_constant<int, 0>());
        step(std::integral_constant<int, 1>());
        step(std::integral_constant<int, 2>());
        step(std::integral_constant<int, 3>());
    };

#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    aim(g0);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) piece(smem, i);
    for (int g = g0; g < g1; ++g) {
        const int odd = (g - g0) & 1;
        stage_barrier();
        if (g + 1 < g1) {
            aim(g + 1);
#pragma unroll
            for (int i = 0; i < PIECES; ++i) piece(smem + (odd ^ 1) * kStage, i);
        }
        compute(smem + odd * kStage);
    }

    const int n = wn * 64 + 2 * l, left = nrows - n, N = (int)p.N;  // 256 rows of up to 2^21 columns: 32 bits hold the offsets
    const int r0 = wm * (TM / WM) + 4 * h;
    if (left <= 0) return;
    float add[2] = {0.f, 0.f};
    if (p.sums == nullptr && p.bias != nullptr) {
        add[0] = p.bias[n0 + n];
        if (left > 1) add[1] = p.bias[n0 + n + 1];
    }
    auto put = [&](auto* to, auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = r0 + i * 32 + (e & 3) + 8 * (e >> 2);
                if (WHOLE || m < mrows) store_two(to, (unsigned)(m * N + n), acc[i][0][e] + add[0], acc[i][1][e] + add[1], WHOLE || left > 1);
            }
    };
    const bool whole = mrows == TM && nrows == TN;
    if (p.sums != nullptr) {
        float* part = p.sums + ((long)split * p.M + m0) * p.N + n0;
        whole ? put(part, std::true_type()) : put(part, std::false_type());
    } else {
        T* out = (T*)p.y + m0 * p.N + n0;
        whole ? put(out, std::true_type()) : put(out, std::false_type());
    }
}

// y = the sum of `splits` fp32 partial results (+ bias of the column)
template <typename T>
__global__ void __launch_bounds__(kT) mx4_join_kernel(const float* __restrict__ sums, int splits, long total, long N, const float* __restrict__ bias,
                                                      T* __restrict__ y) {
    for (long i = blockIdx.x * (long)kT + threadIdx.x; i < total; i += (long)gridDim.x * kT) {
        float v = 0.f;
        for (int s = 0; s < splits; ++s) v += sums[s * total + i];
        if (bias != nullptr) v += bias[i % N];
        store_elem<T>(y, i, v);
    }
}

// dy in the form the gradient's tiles take: `parts` matrices [M][pitch] of 16-bit values, zeros behind the last column.  fp32 is
// cut into three bf16 parts, each the next 8 bits, part p times 2^(kPartUp p) (it meets weights that much smaller): they add up to it
// exactly over all of fp32's range, where plain parts of values below 2^-110 would lose the bits below bf16's last, 2^-133.
// 16-bit types are copied.
constexpr int kPartUp = 8;
template <typename T, int PARTS>
__global__ void __launch_bounds__(kT) mx4_parts_kernel(const T* __restrict__ dy, long ld, long M, long N, long pitch, unsigned short* __restrict__ out) {
    const long total = M * pitch;
    for (long i = blockIdx.x * (long)kT + threadIdx.x; i < total; i += (long)gridDim.x * kT) {
        const long m = i / pitch, n = i - m * pitch;
        if constexpr (PARTS == 1) {
            out[i] = n < N ? reinterpret_cast<const unsigned short*>(dy)[m * ld + n] : 0;
        } else {
            float left = n < N ? load_elem<T>(dy, m * ld + n) : 0.f;
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                const unsigned top = __float_as_uint(left) & 0xffff0000u;  // towards zero: never past the largest number
                out[p * total + i] = (unsigned short)(left != left ? 0x7fc0u : top >> 16);
                left = left != left || __uint_as_float(top) == left ? 0.f : (left - __uint_as_float(top)) * (float)(1 << kPartUp);
            }
        }
    }
}

// dx = dy W for a frozen W: 256 rows x 256 columns (one group of W's) per workgroup of 8 waves, 64 rows of W a step; the only
// tile there is: fewer rows cost what 256 do.  dy comes
// by DMA like the tiles above; W's codes (8 KB a step) are widened to 16 bits on the way into LDS [n][column] and read transposed
// (ds_read_b64_tr_b16), even and odd columns apart as above.  The scale of a weight varies along the sum, so it is applied while
// widening.  bf16 holds every weight as it is (subnormals too, which conversion and products keep), so that sums overflow where the
// result does and not before; raised() says where the weights of 32 columns are moved by a power of two, undone in the end.  fp16
// weights are taken relative to the largest scale of their 32 columns over all rows of W (dy is at most 65504: no sum can overflow), which
// holds scales that are at most 2^26 apart exactly; where a workgroup finds them further apart it cuts each dy value into two bf16
// parts (8 + 3 bits) instead.
// Bound by the 16-bit matrix rate and the widening beside it: 8192 x 8192 x 8192 bf16 967 us, 1.1 PFLOP/s (the library's product of 16-bit
// matrices 1.38); 8192 x 9216 x 9216 fp16 1370 - 1510 us as the card's power allows (matrix units busy 42 % of the cycles, vector units 22 %).
template <typename T, bool CUT>
__device__ __forceinline__ void dgrad_mma(f32x16& acc, const uint4& a, const uint4& b) {
    if constexpr (!CUT) {
        mma32<T>(acc, __builtin_bit_cast(typename MmaFrag<T>::type, a), __builtin_bit_cast(typename MmaFrag<T>::type, b));
    } else {
        float f[8];
        unpack16<_Float16>(a, f);
        bf16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float top = __uint_as_float(__float_as_uint(f[e]) & 0xffff0000u);
            hi[e] = (__bf16)top;
            lo[e] = (__bf16)(top == f[e] ? 0.f : f[e] - top);
        }
        mma32<__bf16>(acc, hi, __builtin_bit_cast(bf16x8, b));
        mma32<__bf16>(acc, lo, __builtin_bit_cast(bf16x8, b));
    }
}

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
template <typename T, int SEL>
__device__ __forceinline__ unsigned widen2(unsigned codes, float scale) {
    if constexpr (__is_same(T, _Float16)) return __builtin_bit_cast(unsigned, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, SEL));
    else return __builtin_bit_cast(unsigned, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL));
}
template <typename T>
__device__ __forceinline__ uint4 widen8(unsigned codes, float scale) {
    return make_uint4(widen2<T, 0>(codes, scale), widen2<T, 1>(codes, scale), widen2<T, 2>(codes, scale), widen2<T, 3>(codes, scale));
}

typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;

// The power of two that bf16 weights of 32 columns are raised by, from their largest E.  Above 252, 6 * 2^(E - 127) is past bf16's
// largest number.  Below 96 there is room: 2^21 products of fp32's largest number stay under 2^121, and the weights that the low
// parts of an fp32 dy meet, smaller by 2^8 and 2^16, stay above the smallest scale.
__device__ __forceinline__ int raised(int emax) { return emax > 252 ? 252 - emax : min(max(96 - emax, 0), 32); }

struct DgradArgs {
    const unsigned char *dy, *codes, *scales;
    long pitch, M, N, width, part_bytes;  // pitch in bytes; width = dy's columns, N (copied: N rounded up to 8); a part = a whole [M][pitch]
    int parts, steps, per_split;   // steps of 64 rows of W, times the parts
    long cols;
    void* dx;
    float* sums;
    unsigned mt, kt;
};

constexpr int kDA = 256 * 128, kDB = 64 * 512;  // bytes of one stage: dy [256][64], W [64][256]

template <typename T, bool CUT>
__device__ __forceinline__ void dgrad_loop(const DgradArgs& p, char* smem, const int* __restrict__ emax, f32x16 (&acc)[4][2], long m0, long g,
                                           int s0, int s1) {
    typedef typename std::conditional<CUT, __bf16, T>::type TW;
    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, l = lane & 31;
    const int nsteps = p.steps / p.parts;
    const long mrows = min(256L, p.M - m0);
    const int row8 = lane >> 3, chunk = (lane & 7) ^ ((w & 1) * 4 + (lane >> 4));
    auto fill_a = [&](int s, char* st) {
        const int part = s / nsteps;
        const long n0 = (s - part * nsteps) * 64L;
        const __amdgpu_buffer_rsrc_t ra = buffer_of(p.dy + part * p.part_bytes + m0 * p.pitch + n0 * 2, (mrows - 1) * p.pitch + (p.width - n0) * 2);
        const bool inside = n0 + chunk * 8 < p.width;  // whole chunks: the width is a multiple of 8
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = (i * 8 + w) * 8;
            lds_dma<16>(ra, st + r * 128, inside ? (int)((r + row8) * p.pitch) + chunk * 16 : (int)0x80000000, 0);
        }
    };
    // a thread takes block kb of one row of W: 16 bytes of codes, one scale
    const int nr = t >> 3, kb = t & 7;
    auto load_b = [&](int s, uint4& c, int& e) {
        const long n = (s % nsteps) * 64L + nr;
        if (n < p.N) {
            c = *reinterpret_cast<const uint4*>(p.codes + (g * p.N + n) * kGroupBytes + kb * 16);
            e = p.scales[(g * p.N + n) * 8 + kb];
        } else {
            c = make_uint4(0, 0, 0, 0);
            e = 0;
        }
    };
    const int add = __is_same(TW, _Float16) ? 140 - emax[kb] : raised(emax[kb]);
    auto store_b = [&](uint4 c, int e, char* st, int part) {
        int x = e == 255 ? 255 : e + add - kPartUp * part;
        if (x < 0) x = 0, c = make_uint4(0, 0, 0, 0);  // below the smallest scale
        const float scale = __uint_as_float(x == 255 ? 0x7fc00000u : (unsigned)x << 23);  // 0 is 2^-127 here; NaN whatever the codes
        // columns 2i and 2i + 1 go to different fragments: the even ones of 64 columns first, then the odd ones, 64 bytes each.
        // Eight of them come from two words of codes in the order 0 4 1 5 2 6 3 7 (out_pair undoes it); which half of the 16 a
        // lane writes first depends on its block, so that a write's sixteen lanes fall on all 64 banks
        const bool second = kb & 4;
        const unsigned x0 = second ? c.z : c.x, y0 = second ? c.w : c.y, x1 = second ? c.x : c.z, y1 = second ? c.y : c.w;
        char* q = st + nr * 512 + (kb & 1) * 32 + (second ? 16 : 0);
        const int even = ((kb & 6) ^ (nr & 3)) << 6, odd = ((kb | 1) ^ (nr & 3)) << 6, other = second ? -16 : 16;
        *reinterpret_cast<uint4*>(q + even) = widen8<TW>((x0 & 0x0f0f0f0fu) | ((y0 & 0x0f0f0f0fu) << 4), scale);
        *reinterpret_cast<uint4*>(q + even + other) = widen8<TW>((x1 & 0x0f0f0f0fu) | ((y1 & 0x0f0f0f0fu) << 4), scale);
        *reinterpret_cast<uint4*>(q + odd) = widen8<TW>(((x0 >> 4) & 0x0f0f0f0fu) | (y0 & 0xf0f0f0f0u), scale);
        *reinterpret_cast<uint4*>(q + odd + other) = widen8<TW>(((x1 >> 4) & 0x0f0f0f0fu) | (y1 & 0xf0f0f0f0u), scale);
    };
    const int wm = w >> 2, wn = w & 3, li = lane & 15, gr = lane >> 4;
    const int brow = (gr >> 1) * 8 + (li >> 2);  // + 16 ks (+ 4): the swizzle depends on the two lowest bits alone
    int boff[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int cb = (wn * 64 + j * 32 + (gr & 1) * 16 + (li & 3) * 4) * 2;
        boff[j] = brow * 512 + ((((cb >> 6) ^ (brow & 3)) << 6) | (cb & 63));
    }
    auto compute = [&](const char* sa, const char* sb, int k0, int k1) {
#pragma unroll
        for (int ks = k0; ks < k1; ++ks) {
            uint4 fa[4], fb[2];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                fa[i] = *reinterpret_cast<const uint4*>(sa + (wm * 128 + i * 32 + l) * 128 + (((ks * 2 + h) ^ ((l >> 1) & 7)) << 4));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const char* q = sb + boff[j] + ks * 16 * 512;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(q));
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(q + 4 * 512));
                fb[j] = __builtin_bit_cast(uint4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) dgrad_mma<T, CUT>(acc[i][j], fa[i], fb[j]);
        }
    };

    uint4 c;
    int e;
    load_b(s0, c, e);
    store_b(c, e, smem + 2 * kDA, s0 / nsteps);
    fill_a(s0, smem);
    load_b(min(s0 + 1, s1 - 1), c, e);
    for (int s = s0; s < s1; ++s) {
        const int cur = (s - s0) & 1;
        const bool more = s + 1 < s1;
        stage_barrier();
        // the codes have arrived with the barrier; naming them here keeps hipcc's own wait for them in front of the requests
        asm volatile("" : "+v"(c.x), "+v"(c.y), "+v"(c.z), "+v"(c.w), "+v"(e));
        if (more) fill_a(s + 1, smem + (cur ^ 1) * kDA);
        compute(smem + cur * kDA, smem + 2 * kDA + cur * kDB, 0, 2);
        if (more) {
            store_b(c, e, smem + 2 * kDA + (cur ^ 1) * kDB, (s + 1) / nsteps);
            load_b(min(s + 2, s1 - 1), c, e);
        }
        compute(smem + cur * kDA, smem + 2 * kDA + cur * kDB, 2, 4);
    }
}
// the pair of columns, of a wave's 32, that lane l ends up with
__device__ __forceinline__ int out_pair(int l) { return (l & 24) + ((l & 7) >> 1) + (l & 1) * 4; }

template <typename T, typename TO>
__global__ void __launch_bounds__(512) mx4_dgrad_kernel(const DgradArgs p) {
    __shared__ __attribute__((aligned(1024))) char smem[2 * (kDA + kDB)];
    __shared__ int emax[8], emin[8];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, h = lane >> 5, l = lane & 31;
    unsigned tm, tk;
    tile_of(xcd_remap(blockIdx.x, gridDim.x), p.mt, p.kt, tm, tk);
    const long m0 = tm * 256L, k0 = tk * 256L, g = tk;
    const int s0 = blockIdx.y * p.per_split, s1 = min(p.steps, s0 + p.per_split);
    // the range of the scales, over all rows of W (a split that covered some of them alone could use a range of its own; the
    // whole range serves every part of dy)
    if (t < 8) emax[t] = 0, emin[t] = 255;
    __syncthreads();
    {
        // two scale bytes per word.  E + 1 and E - 1 modulo 256 leave NaN (255) out of the largest, and E = 0 -- zeros, in all but the
        // smallest of weights -- out of the smallest
        u16x2 hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) hi[i] = 0, lo[i] = 255;
        for (long n = t; n < p.N; n += 512) {
            const uint2 v = *reinterpret_cast<const uint2*>(p.scales + (g * p.N + n) * 8);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned x = ((i < 2 ? v.x : v.y) >> (8 * (i & 1))) & 0x00ff00ffu;
                hi[i] = __builtin_elementwise_max(hi[i], __builtin_bit_cast(u16x2, (x + 0x00010001u) & 0x00ff00ffu));
                lo[i] = __builtin_elementwise_min(lo[i], __builtin_bit_cast(u16x2, (x + 0x00ff00ffu) & 0x00ff00ffu));
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) {
                hi[i] = __builtin_elementwise_max(hi[i], __builtin_bit_cast(u16x2, __shfl_xor(__builtin_bit_cast(int, hi[i]), off, 64)));
                lo[i] = __builtin_elementwise_min(lo[i], __builtin_bit_cast(u16x2, __shfl_xor(__builtin_bit_cast(int, lo[i]), off, 64)));
            }
            const int b = (i >> 1) * 4 + (i & 1);  // bytes b and b + 2
            if (lane == 0) {
                atomicMax(&emax[b], max((int)hi[i].x, 1) - 1), atomicMax(&emax[b + 2], max((int)hi[i].y, 1) - 1);
                atomicMin(&emin[b], lo[i].x + 1), atomicMin(&emin[b + 2], lo[i].y + 1);
            }
        }
    }
    __syncthreads();
    f32x16 acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    bool relative = false;
    if constexpr (__is_same(T, _Float16)) {
        bool wide = false;
        for (int i = 0; i < 8; ++i) wide |= emax[i] - emin[i] > 26;
        if (wide) {
            dgrad_loop<T, true>(p, smem, emax, acc, m0, g, s0, s1);
        } else {
            dgrad_loop<T, false>(p, smem, emax, acc, m0, g, s0, s1);
            relative = true;
        }
    } else {
        dgrad_loop<T, false>(p, smem, emax, acc, m0, g, s0, s1);
    }
    const int wm = w >> 2, wn = w & 3, kc = wn * 64 + 2 * out_pair(l), left = (int)min(256L, p.cols - k0) - kc;
    const int mrows = (int)min(256L, p.M - m0), r0 = wm * 128 + 4 * h, cols = (int)p.cols;
    if (left <= 0) return;
    const int up = relative ? emax[kc >> 5] - 140 : -raised(emax[kc >> 5]);
    auto put = [&](auto* to, auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = r0 + i * 32 + (e & 3) + 8 * (e >> 2);  // 32 bits hold the offsets: cols is at most 2^21
                if (WHOLE || m < mrows)
                    store_two(to, (unsigned)(m * cols + kc), ldexpf(acc[i][0][e], up), ldexpf(acc[i][1][e], up), WHOLE || left > 1);
            }
    };
    const bool whole = mrows == 256 && p.cols - k0 >= 256;
    if (p.sums != nullptr) {
        float* part = p.sums + ((long)blockIdx.y * p.M + m0) * p.cols + k0;
        whole ? put(part, std::true_type()) : put(part, std::false_type());
    } else {
        TO* out = (TO*)p.dx + m0 * p.cols + k0;
        whole ? put(out, std::true_type()) : put(out, std::false_type());
    }
}

long groups_of(long cols) { return (cols + kGroup - 1) / kGroup; }
bool grid_ok(long blocks, int threads = kT) { return blocks > 0 && blocks <= 0xffffffffL / threads; }  // a grid holds fewer than 2^32 threads

// How many parts a sum of `steps` is cut into: at most `most`, and no more than pay for the join, which writes and reads 8 bytes an
// output and part (about 5 TB/s) while a step of a tile takes step_us.  steps step_us / s + s outputs 8 / 5e6 us is smallest at
// s^2 = steps step_us 5e6 / 8 / outputs.
int parts_of(long most, long steps, float step_us, long outputs) {
    long s = 1;
    while (s < most && (s + 1.0) * (s + 1.0) * outputs <= steps * step_us * 625e3) ++s;
    const long per = (steps + s - 1) / s;
    return (int)((steps + per - 1) / per);
}

// How the work of y = a b^T is cut.
struct GemmPlan {
    int tile;        // 0: few rows, straight from memory; else the edge of a square tile
    long mt, nt;
    int splits, per_split;
};
constexpr long kCus = 256;
constexpr int NWR = 8;  // waves that share 16 columns of few rows
// Few rows are multiplied straight from memory up to 32 (16) MB of b: below, tiles cannot fill the machine (4096 x 4096 at 16
// rows 8.9 us, as tiles 14.3; 9216 x 4608 14.7, 17.3); above, DMA reads faster than the waves' own loads (9216 x 9216 at 16 rows 21.5,
// as tiles 19.7; 18432 x 18432 at 2 / 16 / 32 rows 41 / 54 / 74, as tiles 38 / 40 / 42).  From x to y, over weights that are in no cache.
// Tiles of 256 x 256 take a tenth less time than 128 x 128 (4096 x 4096 x 8192: 74 / 81 us, 4096 x 8192 x 8192: 146 / 162) where their
// rounds of 256 are at most 15 % more than their number (8192 x 9216 x 9216, 4.5 rounds: 378 / 401 us), and are slower where the last
// round leaves more idle (4608 x 4096 x 4096, 1.13 rounds: 70 / 58 us; 6144, 1.5 rounds: 73 / 68; 8192 x 5120, 2.5: 112 / 110).
// Sums are cut where tiles are fewer than two workgroups per CU could take (512 x 2048 x 18432: 26 us, 52 in one part;
// 1024 x 2048 x 8192: 24 us in 2 parts, 26 in one, 30 in 4); a part keeps at least 4 steps.
GemmPlan gemm_plan(long M, long N, long G) {
    GemmPlan p = {0, 1, (N + 15) / 16, 1, (int)G};
    if (M <= 32 && N * G * (kGroupBytes + 8) <= (M <= 16 ? 1L << 25 : 1L << 24)) return p;
    const long big = ((M + 255) / 256) * ((N + 255) / 256), rounds = (big + kCus - 1) / kCus;
    p.tile = rounds * kCus * 100 <= big * 115 ? 256 : 128;
    p.mt = (M + p.tile - 1) / p.tile;
    p.nt = (N + p.tile - 1) / p.tile;
    if (p.tile == 128) {
        const long most = 2 * kCus / (p.mt * p.nt);
        p.splits = parts_of(most < G / 4 ? most : G / 4, G, 0.7f, M * N);
        p.per_split = (int)((G + p.splits - 1) / p.splits);
    }
    return p;
}

struct DgradPlan {
    long mt, kt, pitch;  // pitch of the copied parts in elements, 0: dy is taken as it lies
    int parts, steps, splits, per_split;
};
DgradPlan dgrad_plan(int dtype, const void* dy, long ld, long M, long N, long cols) {
    DgradPlan p = {(M + 255) / 256, groups_of(cols), 0, dtype == MSFWSI_DT_F32 ? 3 : 1, 0, 1, 0};
    // DMA takes 16-byte chunks of rows, and a tile's rows lie within 2 GB
    if (dtype == MSFWSI_DT_F32 || N % 8 != 0 || ld % 8 != 0 || ld > (1L << 21) || (reinterpret_cast<uintptr_t>(dy) & 15)) p.pitch = (N + 7) / 8 * 8;
    p.steps = p.parts * (int)((N + 63) / 64);
    p.per_split = p.steps;
    // 512 x 1000 x 512: 20 us, 33 in one part; 256 x 512 x 18432: 22 us in one part, 34 in three
    const long most = kCus / (p.mt * p.kt);
    p.splits = parts_of(most < p.steps / 2 ? most : p.steps / 2, p.steps, 1.6f, M * cols);
    p.per_split = (p.steps + p.splits - 1) / p.splits;
    return p;
}
long round16(long bytes) { return (bytes + 15) / 16 * 16; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
unsigned stride_grid(long items) {
    const long b = (items + kT - 1) / kT;
    return (unsigned)(b > 8 * kCus ? 8 * kCus : b);
}

}  // namespace

#define ST(s) reinterpret_cast<hipStream_t>(s)

extern "C" int msfwsi_mx4_quantize(int dtype, const void* x, long ld, long rows, long cols, void* codes, void* scales, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && rows >= 0 && cols > 0 && (rows <= 1 || ld >= cols));
    if (rows == 0) return MSFWSI_OK;
    const long G = groups_of(cols);
    MSFWSI_CHECK_ARG(x && codes && scales && aligned16(codes) && aligned16(scales) && G <= 65535L * UG && grid_ok((rows + 7) / 8));
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL(mx4_quantize_kernel<T>, dim3((unsigned)((rows + 7) / 8), (unsigned)((G + UG - 1) / UG)), dim3(kT), 0,
                                            ST(stream), (const T*)x, ld, rows, cols, (int)G, (unsigned*)codes, (unsigned*)scales));
    return msfwsi_launch_status();
}

extern "C" int msfwsi_mx4_dequantize(int dtype, const void* codes, const void* scales, long rows, long cols, void* y, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && rows >= 0 && cols > 0);
    if (rows == 0) return MSFWSI_OK;
    const long G = groups_of(cols);
    MSFWSI_CHECK_ARG(y && codes && scales && aligned16(codes) && aligned16(scales) && G <= 65535L * UG && grid_ok((rows + 7) / 8));
    const dim3 grid((unsigned)((rows + 7) / 8), (unsigned)((G + UG - 1) / UG));
#define MX4_WIDEN(T) \
    hipLaunchKernelGGL(mx4_dequantize_kernel<T>, grid, dim3(kT), 0, ST(stream), (const unsigned*)codes, (const unsigned char*)scales, rows, cols, (int)G, (T*)y)
    if (dtype == MSFWSI_DT_F32)
        hipLaunchKernelGGL(mx4_dequantize32_kernel, grid, dim3(kT), 0, ST(stream), (const unsigned short*)codes, (const unsigned char*)scales, rows, cols,
                           (int)G, (float*)y);
    else if (dtype == MSFWSI_DT_BF16) MX4_WIDEN(__bf16);
    else MX4_WIDEN(_Float16);
    return msfwsi_launch_status();
}

extern "C" int msfwsi_mx4_gemm_workspace(long M, long N, long cols, long* bytes) {
    MSFWSI_CHECK_ARG(bytes && M >= 0 && N > 0 && cols > 0 && groups_of(cols) <= 0x7fffffffL);
    const GemmPlan p = gemm_plan(M, N, groups_of(cols));
    *bytes = p.splits > 1 ? p.splits * M * N * 4 : 0;
    return MSFWSI_OK;
}

extern "C" int msfwsi_mx4_gemm(int dtype, const void* a_codes, const void* a_scales, long M, const void* b_codes, const void* b_scales,
                               long N, long cols, const float* bias, void* y, void* workspace, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && M >= 0 && N > 0 && cols > 0);
    if (M == 0) return MSFWSI_OK;
    const long G = groups_of(cols);
    MSFWSI_CHECK_ARG(a_codes && a_scales && b_codes && b_scales && y && G <= 0x7fffffffL);
    MSFWSI_CHECK_ARG(aligned16(a_codes) && aligned16(a_scales) && aligned16(b_codes) && aligned16(b_scales));
    const GemmPlan p = gemm_plan(M, N, G);
    MSFWSI_CHECK_ARG(p.splits == 1 || (workspace && aligned16(workspace)));
    if (N > (1L << 21) || p.mt > 0x7fffffffL || p.nt > 0x7fffffffL || p.nt > 0x7fffffffL / p.mt || !grid_ok(p.mt * p.nt * p.splits, 512)) return MSFWSI_EUNSUPPORTED;
    const unsigned char *a = (const unsigned char*)a_codes, *as = (const unsigned char*)a_scales;
    const unsigned char *b = (const unsigned char*)b_codes, *bs = (const unsigned char*)b_scales;
    const unsigned mt = (unsigned)p.mt, nt = (unsigned)p.nt;
    if (p.tile == 0) {
#define MX4_ROWS(FA)                                                                                                                           \
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL((mx4_gemm_kernel<T, float, false, FA, NWR>), dim3(nt), dim3(NWR * 64), 0, ST(stream), a, as, M, cols, b, \
                                            bs, N, (int)G, bias, (T*)y))
        if (M <= 16) MX4_ROWS(1);
        else MX4_ROWS(2);
        return msfwsi_launch_status();
    }
    float* sums = p.splits > 1 ? (float*)workspace : nullptr;
    GemmArgs args = {a, as, b, bs, M, N, (int)G, p.per_split, bias, y, sums, mt, nt};
    const unsigned grid = mt * nt * p.splits;
#define MX4_TILE(TM, WM, WN) \
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL((mx4_tile_kernel<T, TM, TM, WM, WN>), dim3(grid), dim3(WM * WN * 64), 0, ST(stream), args))
    if (p.tile == 256) MX4_TILE(256, 2, 4);
    else MX4_TILE(128, 2, 2);
    const int rc = msfwsi_launch_status();
    if (rc != MSFWSI_OK || p.splits == 1) return rc;
    MSFWSI_WITH_T(dtype, hipLaunchKernelGGL(mx4_join_kernel<T>, dim3(stride_grid(M * N)), dim3(kT), 0, ST(stream), sums, p.splits, M * N, N, bias, (T*)y));
    return msfwsi_launch_status();
}

// A single row is quantised by the waves that multiply it, in one launch and without a workspace, unless the weight is so large that
// its slower reads cost what the other launches do (from x to y, over weights that are in no cache: 512 x 18432 8.8 us, in more launches
// 10.9; 9216 x 18432 21.6, 25.3; 18432 x 18432 38.1, 37.9)
static bool row_alone(long M, long N, long cols) {
    const long G = groups_of(cols);
    return M == 1 && G <= kRowGroups && N * G * (kGroupBytes + 8) <= 1L << 27;
}
// workspace of a linear call: x's codes, its scales, the partial sums
extern "C" int msfwsi_mx4_linear_workspace(long M, long N, long cols, long* bytes) {
    const int rc = msfwsi_mx4_gemm_workspace(M, N, cols, bytes);
    if (rc == MSFWSI_OK) *bytes = row_alone(M, N, cols) ? 0 : *bytes + groups_of(cols) * M * kGroupBytes + round16(groups_of(cols) * M * 8);
    return rc;
}

template <typename TX>
static void launch_row(int y_dtype, const void* x, const void* codes, const void* scales, long N, long cols, const float* bias, void* y, void* stream) {
    MSFWSI_WITH_T(y_dtype, hipLaunchKernelGGL((mx4_gemm_kernel<T, TX, true, 1, NWR>), dim3((unsigned)((N + 15) / 16)), dim3(NWR * 64), 0, ST(stream), x,
                                              (const unsigned char*)nullptr, 1L, cols, (const unsigned char*)codes, (const unsigned char*)scales, N,
                                              (int)groups_of(cols), bias, (T*)y));
}

extern "C" int msfwsi_mx4_linear(int dtype, const void* x, long ld, long M, const void* codes, const void* scales, long N, long cols,
                                 const float* bias, int y_dtype, void* y, void* workspace, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dtype) && msfwsi_dtype_ok(y_dtype) && M >= 0 && N > 0 && cols > 0);
    if (M == 0) return MSFWSI_OK;
    MSFWSI_CHECK_ARG(codes && scales && y);
    if (row_alone(M, N, cols)) {
        MSFWSI_CHECK_ARG(x && aligned16(codes) && aligned16(scales));
        if (N > (1L << 21)) return MSFWSI_EUNSUPPORTED;
        if (dtype == MSFWSI_DT_BF16) launch_row<__bf16>(y_dtype, x, codes, scales, N, cols, bias, y, stream);
        else if (dtype == MSFWSI_DT_F16) launch_row<_Float16>(y_dtype, x, codes, scales, N, cols, bias, y, stream);
        else launch_row<float>(y_dtype, x, codes, scales, N, cols, bias, y, stream);
        return msfwsi_launch_status();
    }
    MSFWSI_CHECK_ARG(workspace && aligned16(workspace));
    char* xc = (char*)workspace;
    char* xs = xc + groups_of(cols) * M * kGroupBytes;
    const int rc = msfwsi_mx4_quantize(dtype, x, ld, M, cols, xc, xs, stream);
    if (rc != MSFWSI_OK) return rc;
    return msfwsi_mx4_gemm(y_dtype, xc, xs, M, codes, scales, N, cols, bias, y, xs + round16(groups_of(cols) * M * 8), stream);
}

extern "C" int msfwsi_mx4_dgrad_workspace(int dy_dtype, const void* dy, long ld, long M, long N, long cols, long* bytes) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dy_dtype) && bytes && M >= 0 && N > 0 && cols > 0);
    const DgradPlan p = dgrad_plan(dy_dtype, dy, M > 1 ? ld : N, M > 0 ? M : 1, N, cols);
    *bytes = round16(p.parts * M * p.pitch * 2) + (p.splits > 1 ? p.splits * M * cols * 4 : 0);
    return MSFWSI_OK;
}

extern "C" int msfwsi_mx4_dgrad(int dy_dtype, const void* dy, long ld, long M, const void* codes, const void* scales, long N, long cols,
                                int dx_dtype, void* dx, void* workspace, void* stream) {
    MSFWSI_CHECK_ARG(msfwsi_dtype_ok(dy_dtype) && msfwsi_dtype_ok(dx_dtype) && M >= 0 && N > 0 && cols > 0 && (M <= 1 || ld >= N));
    if (M == 0) return MSFWSI_OK;
    MSFWSI_CHECK_ARG(dy && codes && scales && dx && aligned16(codes) && aligned16(scales));
    if (M == 1) ld = N;  // a single row's pitch means nothing
    const DgradPlan p = dgrad_plan(dy_dtype, dy, ld, M, N, cols);
    MSFWSI_CHECK_ARG((p.pitch == 0 && p.splits == 1) || (workspace && aligned16(workspace)));
    if (N > (1L << 21) || cols > (1L << 21) || p.mt > 0x7fffffffL || p.kt > 0x7fffffffL || p.kt > 0x7fffffffL / p.mt || !grid_ok(p.mt * p.kt, 512)) return MSFWSI_EUNSUPPORTED;
    const long copied = p.parts * M * p.pitch * 2;
    if (p.pitch != 0) {
        unsigned short* out = (unsigned short*)workspace;
        if (dy_dtype == MSFWSI_DT_F32)
            hipLaunchKernelGGL((mx4_parts_kernel<float, 3>), dim3(stride_grid(M * p.pitch)), dim3(kT), 0, ST(stream), (const float*)dy, ld, M, N, p.pitch, out);
        else
            hipLaunchKernelGGL((mx4_parts_kernel<__bf16, 1>), dim3(stride_grid(M * p.pitch)), dim3(kT), 0, ST(stream), (const __bf16*)dy, ld, M, N, p.pitch, out);
        const int rc = msfwsi_launch_status();
        if (rc != MSFWSI_OK) return rc;
    }
    DgradArgs d;
    d.dy = p.pitch != 0 ? (const unsigned char*)workspace : (const unsigned char*)dy;
    d.codes = (const unsigned char*)codes;
    d.scales = (const unsigned char*)scales;
    d.pitch = (p.pitch != 0 ? p.pitch : ld) * 2;
    d.M = M;
    d.N = N;
    d.width = p.pitch != 0 ? p.pitch : N;
    d.part_bytes = M * p.pitch * 2;
    d.parts = p.parts;
    d.steps = p.steps;
    d.per_split = p.per_split;
    d.cols = cols;
    d.dx = dx;
    d.sums = p.splits > 1 ? (float*)((char*)workspace + round16(copied)) : nullptr;
    d.mt = (unsigned)p.mt;
    d.kt = (unsigned)p.kt;
    const dim3 grid((unsigned)(p.mt * p.kt), p.splits);
#define MX4_DGRAD(TO)                                                                                                  \
    do {                                                                                                               \
        if (dy_dtype == MSFWSI_DT_F16) hipLaunchKernelGGL((mx4_dgrad_kernel<_Float16, TO>), grid, dim3(512), 0, ST(stream), d); \
        else hipLaunchKernelGGL((mx4_dgrad_kernel<__bf16, TO>), grid, dim3(512), 0, ST(stream), d);                    \
    } while (0)
    if (dx_dtype == MSFWSI_DT_BF16) MX4_DGRAD(__bf16);
    else if (dx_dtype == MSFWSI_DT_F16) MX4_DGRAD(_Float16);
    else MX4_DGRAD(float);
    const int rc = msfwsi_launch_status();
    if (rc != MSFWSI_OK || p.splits == 1) return rc;
    MSFWSI_WITH_T(dx_dtype, hipLaunchKernelGGL(mx4_join_kernel<T>, dim3(stride_grid(M * cols)), dim3(kT), 0, ST(stream), d.sums, p.splits, M * cols, cols,
                                               (const float*)nullptr, (T*)dx));
    return msfwsi_launch_status();
}
