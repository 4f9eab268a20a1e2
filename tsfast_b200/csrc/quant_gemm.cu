// Product with both operands in 8-bit floating point (e4m3) and power-of-two scales:
//   y[m, n] = sum_k deq(x)[m, k] deq(w)[n, k] (+ bias[n]),   x in bfloat16 or float16, y of x's type,
// x quantised here, one scale per row and 128 values; w quantised beforehand, one scale per 128 x 128 block.
// A scale is the smallest power of two s with |v| <= 448 s, so dividing by it is exact and the only rounding is the
// one to e4m3 (to nearest, ties to even); a scale of amax / 448 would round twice and gain nothing, since a floating
// format has the same relative precision at every exponent. A value that is not finite becomes NaN.
//
// The tensor cores multiply e4m3, scale and add in float32: tcgen05.mma.kind::mxf8f6f4 takes a scale (an exponent,
// UE8M0) per 32 values of either operand from tensor memory, and a block of 128 repeats its scale four times. A weight
// scale that is not a power of two has no such exponent: it becomes the exponent code of NaN, and so do the results.
// (Scaling outside, every block's product leaving tensor memory to be added to registers, took 650 us at 8192 x 8192 x
// 4096: 256 columns x 128 lanes per block are as much work for the warps as the block's four MMAs are for the tensor core.)
//
// One CTA makes 128 features x TN tokens: the weights are the operand with 128 rows whatever the number of
// tokens, so a few tokens cost a narrow second operand (TN = 16) instead of a mostly empty tile, and a thread of the
// epilogue owns a feature, so that a warp stores neighbouring features. Warps have fixed roles:
//   warp 0   requests the operands' blocks (TMA, 128-byte swizzle, one block of 128 values per row = one swizzle row) and
//            their scales, 512 bytes per 128 rows
//   warp 1   moves the scales on into tensor memory (tcgen05.cp) and issues the block's four MMAs (K = 32 each), which
//            follow in the same pipe: no warp has to hand anything over between the copies and the product
//   warps 4-11  take the finished accumulator (warp w: lanes 32 (w % 4).., half of the columns) to registers, already
//            in the result's type, give it back and store while the next tile is under way
// Many tokens: a pair of CTAs (cta_group::2) makes 256 features x 256 tokens, and each fetches half of either operand, 33 KB
// per block instead of 49, six of them on their way. One CTA per tile is bound by what it fetches: 258 us at 8192 x 8192 x 4096
// against 221 (2480 TFLOP/s with the quantisation of x, calls one by one; 266 to 284 us, about 2000 TFLOP/s, in a long run of them, where
// the clock falls under the power limit; 200 us remain if x is not fetched, and 181 without any fetching or storing, close to the
// 4 x 128 cycles of a block's MMAs). What issues the MMAs is one elected lane: a lane chosen by its number makes
// the compiler loop over lanes for every instruction, and 263 us.
// Few tiles (small M): a cluster of S CTAs shares a tile, each with its part of K; the parts meet in distributed shared
// memory and are added in the order of the ranks. Every wait on an mbarrier is bounded: one that runs out raises a
// flag that all roles poll, and b200_block_status reports B200_ERR_TIMEOUT.
#include <cuda.h>

#include <type_traits>

#include "block.cuh"

namespace b200 {
namespace quant {

constexpr int kBlock = 128;      // values per scale, bytes per swizzle row
constexpr int kFeatures = 128;   // rows of the first operand
constexpr int kThreads = 384;
constexpr int kStorers = 256;    // threads of warps 4-11
constexpr int kMaxSplit = 8;
constexpr int kWaitLimit = 1 << 18;  // polls of an mbarrier before a wait gives up: about a second, a poll waits 4 us itself

template <int TN, bool PAIR>
struct Shape {
    static constexpr int rows = PAIR ? TN / 2 : TN;  // of the second operand in this CTA's shared memory
    static constexpr int stage = kFeatures * kBlock + rows * kBlock;
    static constexpr int stages = rows == 256 ? 4 : rows == 128 ? 6 : 8;
    static constexpr int x_words = TN <= 128 ? 128 : 256;                   // x's scales of a block, in whole groups of 128 rows
    static constexpr int scale_words = 128 + x_words;                       // and w's before them
    static constexpr int scales = scale_words / 32;  // tensor-memory columns of a block's scales
    static constexpr int cols = TN + stages * scales <= 64 ? 64 : TN + stages * scales <= 128 ? 128 : TN + stages * scales <= 256 ? 256 : 512;
    static constexpr int smem = stages * (stage + scale_words * 4) + 1024;  // operands, then scales
};

// ------------------------------------------------------------------------------------------- quantisation
// exponent of the block's scale from the bits of its largest magnitude: amax = 1.f * 2^k with 448 = 1.75 * 2^8
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t b = __float_as_uint(amax);
    if (b == 0) return 0;
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | (uint32_t)hi << 16;
}
// v times 2^-e; what is not finite becomes NaN (a saturating conversion would make 448 of an infinity)
__device__ __forceinline__ float scaled(float v, float inv) { return fabsf(v) <= 3.402823466e38f ? v * inv : __uint_as_float(0x7fc00000u); }

__device__ __forceinline__ float2 pair_of(uint32_t v, __nv_bfloat16) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
__device__ __forceinline__ float2 pair_of(uint32_t v, __half) {
    __half2 h;
    memcpy(&h, &v, 4);
    return __half22float2(h);
}

// a scale's exponent as UE8M0; the code of NaN for what is not a power of two
__device__ __forceinline__ uint32_t exponent_code(float s) {
    const uint32_t b = __float_as_uint(s), e = b >> 23;
    return (b & 0x7fffffu) != 0 || e == 0 || e > 254 ? 255u : e;
}
// Scales as the product takes them: the exponents (biased by 127) of four consecutive blocks of a row in the bytes of a word
// (an instruction names the byte that it wants), and the words of 128 rows in the order of tensor memory, rows r, r + 32,
// r + 64 and r + 96 side by side. One word per block, its exponent four times: 279 us at 8192 x 8192 x 4096 against 260.
__device__ __forceinline__ long long scale_place(long long row) { return (row & ~127LL) + (row & 31) * 4 + ((row & 127) >> 5); }

// x [M, K] -> q [M, Kp] and scale [groups of four blocks, pitch]. Half a warp has a block of 128, eight values per lane; a warp has four
// blocks of a row, two at a time. Behind these blocks of the grid, others spread the weights' scales in the same way:
// w_words [blocks of features, groups, 128]. The product may be launched at once: it waits for the end of this grid before it
// touches any of the results.
constexpr int kRowBlocks = 4;
template <typename T>
__global__ void __launch_bounds__(256) quant_rows_kernel(const T* __restrict__ x, long long ldx, long long M, int K, int kb, int vec, uint8_t* __restrict__ q,
                                                         uint32_t* __restrict__ scale, long long pitch, const float* __restrict__ sw,
                                                         uint32_t* __restrict__ w_words, long long n_sw, long long x_blocks) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (blockIdx.x >= x_blocks) {
        const long long i = ((long long)blockIdx.x - x_blocks) * 256 + threadIdx.x;  // four words per thread
        if (i < n_sw * 32) {
            const int groups = (kb + kRowBlocks - 1) / kRowBlocks, g = (int)(i / 32 % groups) * kRowBlocks;
            const float* of = sw + i / 32 / groups * kb;
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < kRowBlocks; ++e) w |= (g + e < kb ? exponent_code(__ldg(of + g + e)) : 127u) << 8 * e;
            reinterpret_cast<uint4*>(w_words)[i] = make_uint4(w, w, w, w);
        }
        return;
    }
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, groups = (kb + kRowBlocks - 1) / kRowBlocks;
    const long long row = w / groups;
    if (row >= M) return;
    const int b0 = (int)(w - row * groups) * kRowBlocks + (lane >> 4), at = (lane & 15) * 8;
    uint32_t v[kRowBlocks / 2][4];  // as they are stored, two to a word
#pragma unroll
    for (int i = 0; i < kRowBlocks / 2; ++i) {
        const int k = (b0 + 2 * i) * kBlock + at;
        const T* p = x + row * ldx + k;
        if (vec && k + 8 <= K) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            v[i][0] = u.x, v[i][1] = u.y, v[i][2] = u.z, v[i][3] = u.w;
        } else {
            T t[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = k + e < K ? p[e] : from_float<T>(0.f);
            memcpy(v[i], t, 16);
        }
    }
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < kRowBlocks / 2; ++i) {
        const int b = b0 + 2 * i;
        // The bits of magnitudes are in the order of the magnitudes, infinities and NaN behind the finite ones: two at a time, and
        // no look at single values where the largest is finite (8192 x 1024 x 8192: 97 us, 101 with a test per value).
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) top = __vmaxu2(top, v[i][e] & 0x7fff7fffu);
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, off));
        const uint16_t bits = (uint16_t)max(top >> 16, top & 0xffffu);
        T largest;
        memcpy(&largest, &bits, 2);
        const float m = to_float(largest);
        const int x2 = scale_exponent(m);
        const float inv = pow2(-x2);
        if (b < kb) {
            float2 f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f[e] = pair_of(v[i][e], T());
                f[e] = m <= 3.402823466e38f ? mul2(f[e], make_float2(inv, inv)) : make_float2(scaled(f[e].x, inv), scaled(f[e].y, inv));
            }
            *reinterpret_cast<uint2*>(q + row * ((long long)kb * kBlock) + b * kBlock + at) =
                make_uint2(pack4(f[0].x, f[0].y, f[1].x, f[1].y), pack4(f[2].x, f[2].y, f[3].x, f[3].y));
        }
        codes |= (uint32_t)(x2 + 127) << 16 * i;
    }
    codes |= __shfl_down_sync(0xffffffffu, codes, 16) << 8;  // the other half's blocks lie between
    if (lane == 0) scale[(long long)(b0 / kRowBlocks) * pitch + scale_place(row)] = codes;
}

// one CTA per 128 x 128 block of the weights
template <typename T>
__global__ void __launch_bounds__(256) quant_weight_kernel(const T* __restrict__ w, long long ldw, int N, int K, uint8_t* __restrict__ q, long long ldq,
                                                           float* __restrict__ scale) {
    __shared__ float top[8];
    const int n0 = blockIdx.y * kBlock, k = blockIdx.x * kBlock + (threadIdx.x & 127), half = threadIdx.x >> 7;
    float m = 0.f;
    for (int r = half; r < kBlock; r += 2)
        if (n0 + r < N && k < K) {
            const float v = fabsf(to_float(w[(long long)(n0 + r) * ldw + k]));
            if (v <= 3.402823466e38f) m = fmaxf(m, v);  // what is not finite is lost itself, and sets no scale
        }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, top[i]);
    const int e = scale_exponent(m);
    const float inv = pow2(-e);
    for (int r = half; r < kBlock; r += 2)
        if (n0 + r < N && k < K)
            q[(long long)(n0 + r) * ldq + k] = (uint8_t)pack4(scaled(to_float(w[(long long)(n0 + r) * ldw + k]), inv), 0.f, 0.f, 0.f);
    if (threadIdx.x == 0) scale[(long long)blockIdx.y * gridDim.x + blockIdx.x] = pow2(e);
}

// ------------------------------------------------------------------------------------------- the product
struct Args {
    void* y;
    long long ldy, M;
    int N, nkb, groups;  // blocks of K, and words of scales for them
    const uint32_t* sx;  // [groups, pitch]
    long long pitch;
    const uint32_t* sw;  // [ceil(N / 128), groups, 128]
    const void* bias;
    int bias_f32;
    int split;        // CTAs of a cluster, each with its part of K
    int polls;        // of a wait
    long long mute;   // a tile whose end is not reported (-1: none)
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) {  // an address in the cluster
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}
// the same, counted on a barrier of the pair's first CTA (`bar` is its address in the cluster)
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, int bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
                 "r"(smem_u32(bar))
                 : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    if constexpr (PAIR)  // the barriers of both CTAs
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                     "h"((uint16_t)3)
                     : "memory");
    else asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint64_t operand(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// D float32, A and B e4m3, both K-major, scales UE8M0 (byte `which` of their words), M = 128 per CTA, N = TN
template <int TN, bool PAIR>
__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t scale_a, uint32_t scale_b, uint32_t which, uint32_t accumulate) {
    const uint32_t idesc = which << 4 | which << 29 | ((uint32_t)(TN >> 3) << 17) | (1u << 23) | ((uint32_t)((PAIR ? 2 * kFeatures : kFeatures) >> 4) << 24);
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)
            : "memory");
    else asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)
        : "memory");
}
// 128 scales from shared memory (32 rows of 16 bytes) to four columns, the same in every quarter of the lanes
template <bool PAIR>
__device__ __forceinline__ void scales_to_tmem(uint32_t at, uint32_t saddr) {
    // rows of 16 bytes, unswizzled, groups of 8 rows 128 bytes apart
    const uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
    if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(at), "l"(d) : "memory");  // in both CTAs
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(at), "l"(d) : "memory");
}
// 8 or 16 consecutive columns of this thread's lane
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// address in the cluster of what the CTA `rank` has at this place
__device__ __forceinline__ uint32_t at_rank(const void* local, int rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
    return a;
}
__device__ __forceinline__ float4 remote(const float* local, int rank) {
    uint32_t a;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}

__device__ unsigned int product_lost;  // B200_ERR_TIMEOUT once a wait ran out

// One lane of a converged warp; the compiler knows that it is one, and issues its tensor-core instructions without a loop over lanes.
__device__ __forceinline__ bool elected() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(one));
    return one != 0;
}

struct NoMap {};
template <bool PAIR>
using ScaleMap = std::conditional_t<PAIR, CUtensorMap, NoMap>;

template <typename T, int TN, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
quant_gemm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ ScaleMap<PAIR> map_sw,
                  const __grid_constant__ ScaleMap<PAIR> map_sx, const Args p) {
    using S = Shape<TN, PAIR>;
    constexpr int HC = TN / 2, PIECE = HC < 16 ? 8 : 16;  // columns per storing thread, and per tensor-memory load
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full[S::stages], empty[S::stages], acc_full, acc_empty;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    const int tid = threadIdx.x, wid = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);

    uint32_t* const scales_in = reinterpret_cast<uint32_t*>(base + S::stages * S::stage);
    if (tid == 0) {
        for (int s = 0; s < S::stages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
        mbar_init(&acc_full, 1), mbar_init(&acc_empty, PAIR ? 2 * kStorers / 32 : kStorers / 32);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (wid == 2) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(S::cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(S::cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if constexpr (PAIR) cluster_sync();
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot, tmem_scales = tmem + TN;

    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        const uint32_t a = smem_u32(bar);
        for (int i = 0; i < p.polls; ++i) {
            uint32_t ok;
            if constexpr (PAIR)
                asm volatile(
                    "{\n\t.reg .pred p;\n\t"
                    "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                    "selp.u32 %0, 1, 0, p;\n\t}"
                    : "=r"(ok)
                    : "r"(a), "r"(parity)
                    : "memory");
            else asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                "selp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(ok)
                : "r"(a), "r"(parity)
                : "memory");
            if (ok) return true;
            if (abort_flag) return false;
        }
        abort_flag = 1;
        return false;
    };

    // a pair's tiles are 256 features wide, 128 in either CTA
    constexpr int kWide = PAIR ? 2 * kFeatures : kFeatures;
    const int member = PAIR ? (int)(blockIdx.x & 1) : 0;
    const int rank = PAIR ? 0 : (int)(blockIdx.x % p.split);
    const long long n_tiles = (p.N + kWide - 1) / kWide, tiles = n_tiles * ((p.M + TN - 1) / TN);
    const int ctas = PAIR ? 2 : p.split;
    const long long t0 = blockIdx.x / ctas, dt = gridDim.x / ctas;
    const int kb0 = (int)((long long)p.nkb * rank / p.split), kb1 = (int)((long long)p.nkb * (rank + 1) / p.split);

    // a block that brings its group's scales
    auto first = [&](int kb) { return kb == kb0 || kb % kRowBlocks == 0; };

    if (wid == 0) {
        if (elected()) {
            int s = 0, done = 0;
            uint32_t phase = 1;  // of `empty`: a fresh barrier passes the wait for the phase before its first
            // in a pair the first CTA's barrier counts both CTAs' copies
            auto fetch = [&](void* dst, const CUtensorMap* map, int x, int y, int s) {
                if constexpr (PAIR) tma_load_pair(dst, map, x, y, at_rank(&full[s], 0));
                else tma_load_2d(dst, map, x, y, &full[s]);
            };
            auto weights = [&](int kb, int n0, int s) {
                if (member == 0) mbar_expect_tx(&full[s], (S::stage + (first(kb) ? S::scale_words * 4 : 0)) * (PAIR ? 2 : 1));
                fetch(base + s * S::stage, &map_w, kb * kBlock, n0, s);
            };
            // the weights do not wait for the rows' quantisation
            const int early = t0 < tiles ? min(S::stages, kb1 - kb0) : 0;
            for (int i = 0; i < early; ++i) weights(kb0 + i, (int)(t0 % n_tiles) * kWide + member * kFeatures, i);
            asm volatile("griddepcontrol.wait;" ::: "memory");
            for (long long t = t0; t < tiles && !abort_flag; t += dt) {
                const long long nt = PAIR ? t % n_tiles * 2 + member : t % n_tiles;
                const int n0 = (int)nt * kFeatures, m0 = (int)(t / n_tiles) * TN;
                const uint32_t* sw = p.sw + nt * p.groups * 128;
                const uint32_t* sx = p.sx + (m0 & ~127);  // of whole groups of 128 rows
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (done >= early) {
                        if (!wait(&empty[s], phase)) break;
                        weights(kb, n0, s);
                    }
                    ++done;
                    fetch(base + s * S::stage + kFeatures * kBlock, &map_x, kb * kBlock, m0 + member * S::rows, s);
                    if (first(kb)) {
                        const int g = kb / kRowBlocks;
                        if constexpr (PAIR) {
                            fetch(scales_in + s * S::scale_words, &map_sw, 0, (int)nt * p.groups + g, s);
                            fetch(scales_in + s * S::scale_words + 128, &map_sx, m0, g, s);
                        } else {
                            bulk_load(scales_in + s * S::scale_words, sw + g * 128, 512, &full[s]);
                            bulk_load(scales_in + s * S::scale_words + 128, sx + g * p.pitch, S::x_words * 4, &full[s]);
                        }
                    }
                    if (++s == S::stages) s = 0, phase ^= 1u;
                }
            }
        }
    } else if (wid == 1) {
        if (member == 0 && elected()) {  // a pair's first CTA issues for both
            int s = 0;
            uint32_t phase = 0, turn = 1, sa = 0;
            for (long long t = t0; t < tiles && !abort_flag; t += dt, turn ^= 1u) {
                bool fine = wait(&acc_empty, turn);
                // a tile of 64 tokens may be the second half of a group of 128 scales
                const uint32_t group = TN == 64 ? (uint32_t)(t / n_tiles & 1) * 2u : 0u;
                for (int kb = kb0; kb < kb1 && fine; ++kb) {
                    if (!wait(&full[s], phase)) {
                        fine = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t st = smem_u32(base + s * S::stage);
                    const uint32_t scales = smem_u32(scales_in + s * S::scale_words);
                    if (first(kb)) {
                        sa = tmem_scales + (uint32_t)(s * S::scales);
#pragma unroll
                        for (int j = 0; j < S::scale_words / 128; ++j) scales_to_tmem<PAIR>(sa + (uint32_t)(4 * j), scales + 512 * j);
                    }
                    const uint64_t a = operand(st), b = operand(st + kFeatures * kBlock);
#pragma unroll
                    for (int k = 0; k < 4; ++k)  // 32 values = 32 bytes along K: +2 in 16-byte units
                        umma<TN, PAIR>(tmem, a + (uint64_t)(2 * k), b + (uint64_t)(2 * k), sa, sa + 4 + group, (uint32_t)(kb % kRowBlocks), (kb != kb0) | (k != 0));
                    umma_commit<PAIR>(&empty[s]);
                    if (++s == S::stages) s = 0, phase ^= 1u;
                }
                if (!fine) break;
                if (t != p.mute) umma_commit<PAIR>(&acc_full);
            }
        }
    } else if (wid >= 4) {
        const int quarter = wid & 3, half = (wid - 4) >> 2;
        const uint32_t column0 = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * HC);
        long long ti = 0;
        for (long long t = t0; t < tiles; t += dt, ++ti) {
            const int n = (int)(t % n_tiles) * kWide + member * kFeatures + quarter * 32 + lane;
            const long long m0 = t / n_tiles * TN + half * HC;
            const float bias = p.bias == nullptr || n >= p.N || p.split > 1 ? 0.f
                               : p.bias_f32                                ? static_cast<const float*>(p.bias)[n]
                                                                           : to_float(static_cast<const T*>(p.bias)[n]);
            // the warp leaves as one: the loads from tensor memory want all of its lanes, and lanes may see the flag at different polls
            if (!__all_sync(0xffffffffu, wait(&acc_full, (uint32_t)(ti & 1)))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float* part = reinterpret_cast<float*>(base);  // (clusters) where the operands' blocks were: all of them have been read
            T out[HC];
#pragma unroll
            for (int c = 0; c < HC; c += PIECE) {
                uint32_t r[PIECE];
                tmem_ld(column0 + (uint32_t)c, r);
                tmem_wait();
                if (!PAIR && p.split > 1) {
#pragma unroll
                    for (int j = 0; j < PIECE; ++j) part[(half * HC + c + j) * kFeatures + quarter * 32 + lane] = __uint_as_float(r[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < PIECE; ++j) out[c + j] = from_float<T>(__uint_as_float(r[j]) + bias);
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {  // all in registers: the next tile may have the accumulator
                if constexpr (PAIR) mbar_arrive_at(at_rank(&acc_empty, 0));
                else mbar_arrive(&acc_empty);
            }
            if ((PAIR || p.split == 1) && n < p.N) {
                T* y = static_cast<T*>(p.y) + m0 * p.ldy + n;
                const long long left = p.M - m0;
#pragma unroll
                for (int c = 0; c < HC; ++c)
                    if (c < left) y[(long long)c * p.ldy] = out[c];
            }
        }
    }
    __syncwarp();
    if (!PAIR && p.split > 1) {
        cluster_sync();
        if (wid >= 4) {
            // a warp adds a token's 128 features, four per lane; all parts are on their way before the first is added
            const int f = 4 * lane, n = (int)(t0 % n_tiles) * kFeatures + f;
            const long long m0 = t0 / n_tiles * TN;
            const float* part = reinterpret_cast<const float*>(base);
            float bias[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                bias[e] = p.bias == nullptr || n + e >= p.N ? 0.f
                          : p.bias_f32                      ? static_cast<const float*>(p.bias)[n + e]
                                                            : to_float(static_cast<const T*>(p.bias)[n + e]);
            for (int c = rank + p.split * (wid - 4); c < TN && m0 + c < p.M; c += 8 * p.split) {
                float4 v[kMaxSplit];
#pragma unroll
                for (int k = 0; k < kMaxSplit; ++k)
                    if (k < p.split) v[k] = remote(part + c * kFeatures + f, k);
                float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < kMaxSplit; ++k)
                    if (k < p.split) s[0] += v[k].x, s[1] += v[k].y, s[2] += v[k].z, s[3] += v[k].w;
                T* y = static_cast<T*>(p.y) + (m0 + c) * p.ldy + n;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < p.N) y[e] = from_float<T>(s[e] + bias[e]);
            }
        }
        cluster_sync();  // nobody leaves while its part is being read
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (abort_flag) {  // (whoever gave up, all of the block are here, and see it)
        if (tid == 0) {
            atomicExch(&product_lost, (unsigned int)B200_ERR_TIMEOUT);
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // copies in flight get a bounded time to land
        }
        __syncthreads();
    }
    if constexpr (PAIR) {
        cluster_sync();  // neither leaves while the other's barriers or blocks are in use
        if (wid == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::cols) : "memory");
    } else if (wid == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::cols) : "memory");
}

// ------------------------------------------------------------------------------------------- host
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode() {
    static EncodeFn fn = nullptr;
    if (fn == nullptr) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeFn>(p);
    }
    return fn;
}
// [rows, cols] scales (32-bit words) in boxes of one row
static bool make_scale_map(CUtensorMap* map, const void* ptr, long long rows, long long cols, int box) {
    EncodeFn fn = encode();
    if (fn == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {4 * (cuuint64_t)cols};
    const cuuint32_t extent[2] = {(cuuint32_t)box, 1}, steps[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(ptr), dims, strides, extent, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// [rows, cols] bytes with a row pitch, in boxes of 128 bytes x `box` rows
static bool make_map(CUtensorMap* map, const void* ptr, long long rows, long long cols, long long pitch, int box) {
    EncodeFn fn = encode();
    if (fn == nullptr) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)pitch};
    const cuuint32_t extent[2] = {kBlock, (cuuint32_t)box}, steps[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, extent, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan {
    int nkb, groups;
    long long pitch;  // of x's scales: whole tiles, so that a tile's scales are copied without a look at M
    size_t sx, sw, q, total;
};
static Plan plan(long long M, long long N, long long K) {
    Plan w;
    w.nkb = (int)((K + kBlock - 1) / kBlock);
    w.groups = (w.nkb + kRowBlocks - 1) / kRowBlocks;
    w.sx = 0;
    w.pitch = (M + 255) / 256 * 256;
    w.sw = align_up(w.sx + sizeof(uint32_t) * (size_t)(w.groups * w.pitch), 256);
    w.q = align_up(w.sw + 512 * (size_t)(w.groups * ((N + kFeatures - 1) / kFeatures)), 1024);
    w.total = w.q + (size_t)M * w.nkb * kBlock;
    return w;
}

template <typename T, int TN, bool PAIR>
int launch_gemm(const CUtensorMap& mw, const CUtensorMap& mx, const ScaleMap<PAIR>& msw, const ScaleMap<PAIR>& msx, Args p, cudaStream_t st) {
    constexpr int kWide = PAIR ? 2 * kFeatures : kFeatures;
    const long long n_tiles = (p.N + kWide - 1) / kWide, tiles = n_tiles * ((p.M + TN - 1) / TN);
    // a tile's K is shared by as many CTAs as fill the device once, two blocks each at least
    p.split = 1;
    while (!PAIR && p.split < kMaxSplit && tiles * (p.split + 1) <= 148 && p.nkb / (p.split + 1) >= 2) ++p.split;
    const long long ctas = PAIR ? 2 : p.split, grid = tiles * ctas < 148 || p.split > 1 ? tiles * ctas : 148;
    const auto kernel = quant_gemm_kernel<T, TN, PAIR>;
    constexpr int smem = Shape<TN, PAIR>::smem;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return B200_ERR_LAUNCH;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned int)grid), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned int)ctas, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, mw, mx, msw, msx, p) == cudaSuccess ? B200_OK : B200_ERR_LAUNCH;
}

template <typename T>
int run(const void* x, long long ldx, const void* q, long long ldq, const float* scale, int K, const Plan& w, char* ws, Args& p, cudaStream_t st) {
    uint32_t* sx = reinterpret_cast<uint32_t*>(ws + w.sx);
    uint8_t* xq = reinterpret_cast<uint8_t*>(ws + w.q);
    uint32_t* sw = reinterpret_cast<uint32_t*>(ws + w.sw);
    p.sx = sx, p.sw = sw, p.pitch = w.pitch, p.nkb = w.nkb, p.groups = w.groups;
    const long long x_blocks = (p.M * w.groups + 7) / 8, n_sw = (long long)w.groups * ((p.N + kFeatures - 1) / kFeatures), blocks = x_blocks + (n_sw + 7) / 8;
    if (blocks > 0x7fffffffLL) return B200_ERR_UNSUPPORTED;
    const int vec = (uintptr_t)x % 16 == 0 && ldx % 8 == 0;
    quant_rows_kernel<T><<<(unsigned int)blocks, 256, 0, st>>>(static_cast<const T*>(x), ldx, p.M, K, w.nkb, vec, xq, sx, w.pitch, scale, sw, n_sw, x_blocks);
    if (cudaGetLastError() != cudaSuccess) return B200_ERR_LAUNCH;
    // Few tokens: the narrowest tile that takes them. More: the narrowest that leaves half the device to splitting K (300 x 520 x
    // 1111: 10.7 us with 64 tokens per tile, 14.8 with 256), or 256, which reads the weights least often (1024 x 4096 x 4096: 31 us
    // against 66 with 64).
    int TN = p.M <= 16 ? 16 : p.M <= 32 ? 32 : p.M <= 64 ? 64 : p.M <= 128 ? 128 : 64;
    while (p.M > 128 && TN < 256 && (p.N + kFeatures - 1) / kFeatures * ((p.M + TN - 1) / TN) > 74) TN *= 2;
    // Pairs of CTAs where K is not split, unless an odd number of feature tiles costs them a turn of the device (8192 x 1152 x 4096:
    // 70 us with pairs, 68 without; 8192 x 2048 x 2048: 52 and 74).
    const long long n_tiles = (p.N + kFeatures - 1) / kFeatures, m_tiles = (p.M + TN - 1) / TN;
    const bool pair = TN == 256 && n_tiles * m_tiles > 74 && ((n_tiles + 1) / 2 * m_tiles + 73) / 74 <= (n_tiles * m_tiles + 147) / 148;
    CUtensorMap mw, mx;
    if (!make_map(&mw, q, p.N, K, ldq, kFeatures) || !make_map(&mx, xq, p.M, (long long)w.nkb * kBlock, (long long)w.nkb * kBlock, pair ? TN / 2 : TN))
        return B200_ERR_LAUNCH;
    if (pair) {
        CUtensorMap msw, msx;
        if (!make_scale_map(&msw, sw, n_tiles * w.groups, 128, 128) || !make_scale_map(&msx, sx, w.groups, w.pitch, 256)) return B200_ERR_LAUNCH;
        return launch_gemm<T, 256, true>(mw, mx, msw, msx, p, st);
    }
    if (TN == 16) return launch_gemm<T, 16, false>(mw, mx, {}, {}, p, st);
    if (TN == 32) return launch_gemm<T, 32, false>(mw, mx, {}, {}, p, st);
    if (TN == 64) return launch_gemm<T, 64, false>(mw, mx, {}, {}, p, st);
    if (TN == 128) return launch_gemm<T, 128, false>(mw, mx, {}, {}, p, st);
    return launch_gemm<T, 256, false>(mw, mx, {}, {}, p, st);
}

int product_status(cudaStream_t st) { return take_error_word(product_lost, st); }

}  // namespace quant
}  // namespace b200

extern "C" {

int b200_quant_weight(int dtype, int64_t N, int64_t K, const void* w, int64_t ldw, void* q, int64_t ldq, void* scale, void* stream) {
    using namespace b200;
    using namespace b200::quant;
    if (block_elem_size(dtype) == 0 || N < 1 || K < 1 || N > (1 << 22) || K > (1 << 22) || !w || !q || !scale || ldw < 0 || ldq < K) return B200_ERR_ARG;
    if (!on_boundary(block_elem_size(dtype), w) || !on_boundary(4, scale)) return B200_ERR_ARG;
    const dim3 grid((unsigned int)((K + kBlock - 1) / kBlock), (unsigned int)((N + kBlock - 1) / kBlock));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == B200_F32) quant_weight_kernel<float><<<grid, 256, 0, st>>>((const float*)w, ldw, (int)N, (int)K, (uint8_t*)q, ldq, (float*)scale);
    else if (dtype == B200_BF16)
        quant_weight_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>((const __nv_bfloat16*)w, ldw, (int)N, (int)K, (uint8_t*)q, ldq, (float*)scale);
    else quant_weight_kernel<__half><<<grid, 256, 0, st>>>((const __half*)w, ldw, (int)N, (int)K, (uint8_t*)q, ldq, (float*)scale);
    return cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_LAUNCH;
}

size_t b200_quant_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0) return 256;
    return b200::quant::plan(M, N, K).total;
}

int b200_quant_probe(int polls, int64_t mute_tile, int dtype, int64_t M, int64_t N, int64_t K, const void* x, int64_t ldx, const void* q, int64_t ldq,
                     const void* scale, const void* bias, int bias_f32, void* y, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace b200;
    using namespace b200::quant;
    if ((dtype != B200_BF16 && dtype != B200_F16) || M < 0 || N < 1 || K < 1 || N > (1 << 22) || K > (1 << 22) || M > 0x7fffff00LL) return B200_ERR_ARG;
    if (M == 0) return B200_OK;
    if (!x || !q || !scale || !y || ldx < 0 || ldy < N || ldq < K || ldq % 16 || (uintptr_t)q % 16 || (uintptr_t)x % 2 || (uintptr_t)y % 2) return B200_ERR_ARG;
    if (!on_boundary(4, scale) || !on_boundary(bias_f32 ? 4 : 2, bias)) return B200_ERR_ARG;
    const Plan w = plan(M, N, K);
    if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < w.total) return B200_ERR_WORKSPACE;
    Args p = {};
    p.y = y, p.ldy = ldy, p.M = M, p.N = (int)N, p.bias = bias, p.bias_f32 = bias_f32;
    p.polls = polls > 0 && polls < kWaitLimit ? polls : kWaitLimit, p.mute = mute_tile;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == B200_BF16 ? run<__nv_bfloat16>(x, ldx, q, ldq, (const float*)scale, (int)K, w, (char*)workspace, p, st)
                              : run<__half>(x, ldx, q, ldq, (const float*)scale, (int)K, w, (char*)workspace, p, st);
}

int b200_quant_linear(int dtype, int64_t M, int64_t N, int64_t K, const void* x, int64_t ldx, const void* q, int64_t ldq, const void* scale,
                      const void* bias, int bias_f32, void* y, int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
    return b200_quant_probe(0, -1, dtype, M, N, K, x, ldx, q, ldq, scale, bias, bias_f32, y, ldy, workspace, workspace_bytes, stream);
}

}  // extern "C"
