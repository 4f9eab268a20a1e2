// The norms around a gated block, one pass over HBM each way (float32, bfloat16, float16 rows; float32 inside):
//   m   = n(x) w1 (+ b1)        (POST; else m = x)         n(v) = (v - mean) / sqrt(var + eps), without the mean for RMS
//   m  *= act(gate)             (optional)
//   res'= residual + scale m    (RES; scale optional)
//   y   = n(res') w2 (+ b2)     (RES; else y = m)
// RES false is the gated norm that closes a block's inner path, RES true is the seam between two blocks.
//
// What bounds the kernels is HBM traffic (every tensor crosses it once) and, for few rows, the latency of the row sums (at
// most two after one another). Rows up to 256 wide belong to 8, 16 or 32 lanes of a warp, wider ones to a CTA of 64 to
// 512 threads, with 4, 8 or 16 columns per thread: always the same ones, so that a thread copies its own pieces of the
// coming rows into shared memory (cp.async, no barrier), keeps its parameters there in float32 and its columns' sums in
// registers. Arithmetic is on pairs (two float32 operations per instruction). All sums are float32; y is taken from the
// unrounded res', and the adjoint recomputes res' from its parts instead of reading the rounded one, so every result is
// rounded once. Column gradients: a CTA writes one partial row, and the rows are added in a fixed order.
//
// Measured (forward and adjoint; every tensor counted once): residual RMS norm 16384 x 4096 bfloat16 115 and 239 us (5.8 and 4.5
// TB/s), 65536 x 1024 113 and 205 us (5.9 and 5.2 TB/s), float32 8192 x 4096 121 and 203 us (5.5 and 5.3 TB/s); gated layer norm
// 256000 x 128 float32 73 and 114 us (5.4 and 5.8 TB/s). Rows off the boundaries cost more (8190 x 1003
// float16: 23 and 38 us; 1024 wide: 12 and 25), and so does the adjoint above 4096 columns, where a thread has 16 columns and an
// SM one CTA (8192 x 8192 bfloat16: 126 and 415 us).
#pragma once
#include "block.cuh"

namespace b200 {
namespace norm {

constexpr int kMaxWidth = 8192;
constexpr int kWarpThreads = 128;  // threads of a CTA whose rows belong to warps
enum { kActNone = 0, kActSilu = 1, kActSigmoid = 2 };
enum { kGW2 = 0, kGScale = 1, kGW1 = 2, kGB2 = 3, kGB1 = 4 };  // parameters and their gradients; the biases come last (mean kinds only)

struct Args {
    long long M;
    int D;
    const void *x, *gate, *res;      // rows with pitches ldx, ldg, ldr; gate may be null
    long long ldx, ldg, ldr;
    const void* par[5];              // [D]; of the rows' type, or float32 (pf32); null: one, or zero for a bias
    int pf32, act;
    float eps;
    void *y, *res_out;               // dense (forward)
    float* stats;                    // [M][4]: mean and 1/std of x, of res'; null: not kept (forward)
    const void *gy, *gres;           // upstream, pitches ldgy, ldgr; gres may be null (adjoint)
    long long ldgy, ldgr;
    void *gx, *ggate, *gresid;       // dense; gx, ggate null: not wanted (adjoint)
    float* part;                     // [CTAs][sums][D] (adjoint)
    int pvec;                        // every parameter starts on the boundary of a thread's piece
    int lanes;                       // lanes per row where rows belong to warps
};

// A thread's E columns of a row come in pieces of up to 16 bytes, G pieces apart, where every row starts on such a boundary
// (AL); else in words of four bytes, G words apart: a warp's accesses are contiguous either way. A 16-bit row may then start in
// the middle of a word; its pairs are put together from two.
template <typename T, int E, bool AL>
struct Piece {
    static constexpr int bytes = !AL ? 4 : E * (int)sizeof(T) < 16 ? E * (int)sizeof(T) : 16;
    static constexpr int cols = bytes / (int)sizeof(T), count = E / cols;
    // of a ring's row: off the boundaries a group of up to 32 lanes keeps a piece of 16 bytes more than its words fill
    static constexpr int row = AL ? count * bytes : E == 4 ? count * 6 : count * 9 / 2;
};
template <typename T, int E, bool AL>
struct Columns {
    using P = Piece<T, E, AL>;
    int t, G, D;
    __device__ __forceinline__ int first(int k) const { return (t + G * k) * P::cols; }
    __device__ __forceinline__ int at(int i) const { return first(i / P::cols) + i % P::cols; }
    // one for columns inside the row, zero past its end
    __device__ __forceinline__ float2 inside(int j) const { return make_float2(at(2 * j) < D ? 1.f : 0.f, at(2 * j + 1) < D ? 1.f : 0.f); }
};

__device__ __forceinline__ float2 pair_of_word(uint32_t v, __nv_bfloat16) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
__device__ __forceinline__ float2 pair_of_word(uint32_t v, __half) {
    __half2 h;
    memcpy(&h, &v, 4);
    return __half22float2(h);
}

// What a thread keeps in shared memory: the rows on their way or at work (three stages, two, or none where not even two
// fit: rows are then loaded when they are worked on) and, where they fit beside those, its parameters.
template <typename T, bool LAYER, bool RES, bool WARP, int E, bool AL, bool BWD>
struct Keeps {
    static constexpr int tensors = BWD ? (RES ? 5 : 3) : (RES ? 3 : 2), params = LAYER ? 5 : 3;
    // bytes per thread: 227 KB for one CTA of 512, or for two where the forward's registers allow them, unless float32 off the
    // boundaries, whose arithmetic is less and whose third stage is worth more (60000 x 997: 269 us with it, 304 with two CTAs;
    // 16383 x 4095 bfloat16: 277 and 230)
    static constexpr int limit = !BWD && !WARP && E <= 8 && (AL || sizeof(T) == 2) ? 220 : 450;
    static constexpr int row = tensors * Piece<T, E, AL>::row, par = params * E * 4;
    static constexpr bool kept = par + 2 * row <= limit;
    static constexpr int stages = (kept ? par : 0) + 3 * row <= limit ? 3 : (kept ? par : 0) + 2 * row <= limit ? 2 : 0;
    static constexpr int bytes = (kept ? par : 0) + stages * row;
};

// The coming rows of N tensors. Slot (stage, tensor, piece) holds a piece per thread, side by side (AL). Off the boundaries a
// slot holds a group's 128 contiguous bytes (of the 32 lanes' words; less where a row has fewer lanes) as the 16-byte pieces of
// memory that they lie in, one more than they fill: the group's lanes fetch them together and read each other's, so a warp
// waits for its lanes before it reads and before it fetches again (`together`). A piece may begin before its row, and never
// leaves the aligned 16 bytes that the row's first or last value lies in. (Words of four bytes, fetched by the thread that
// needs them, two for a pair across a boundary: 8190 x 1003 float16 27 and 49 us against 23
// and 38; stores in whole words, put together from two lanes, changed nothing.)
template <typename T, int E, bool AL, int N>
struct Ring {
    using P = Piece<T, E, AL>;
    unsigned char* base;  // slot 0 of this thread (AL) or of its group
    int pitch;            // bytes of a slot: all threads' pieces
    static __device__ __forceinline__ int lanes(const Columns<T, E, AL>& c) { return E > 4 || c.G > 32 ? 32 : c.G; }
    static __device__ __forceinline__ Ring at(const Columns<T, E, AL>& c, unsigned char* mem) {
        if constexpr (AL) {
            return {mem + threadIdx.x * P::bytes, (int)blockDim.x * P::bytes};
        } else {
            const int lw = lanes(c), bytes = 4 * lw + 16;
            return {mem + threadIdx.x / lw * bytes, (int)blockDim.x / lw * bytes};
        }
    }
    static __device__ __forceinline__ void together() {
        if constexpr (!AL) __syncwarp();
    }
    __device__ __forceinline__ unsigned char* slot(int stage, int q, int k) const { return base + ((stage * N + q) * P::count + k) * pitch; }
    template <int B>
    static __device__ __forceinline__ void fetch(unsigned char* to, const void* from, int n) {  // n bytes of B, the others zero
        const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
        if constexpr (B == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from), "r"(n) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(at), "l"(from), "r"(n), "n"(B) : "memory");
    }
    __device__ __forceinline__ void copy(const Columns<T, E, AL>& c, int stage, int q, const void* src, long long offset) const {
        const T* row = static_cast<const T*>(src) + offset;
        if constexpr (AL) {
#pragma unroll
            for (int k = 0; k < P::count; ++k) {
                // Nothing is read of a piece behind the row. How its unused address is written decides how the compiler schedules the
                // loop: rounded down, the adjoint of float32 rows of one piece per thread takes 115 us instead of 132 (256000 x 128),
                // but the others are slower (16384 x 4096 bfloat16: 255 us against 239).
                const int col = c.first(k), left = c.D - col;
                const T* from = row + (left > 0 ? col : 0);
                if constexpr (E == 4 && sizeof(T) == 4) from = left > 0 ? from : reinterpret_cast<const T*>((uintptr_t)from & ~(uintptr_t)15);
                fetch<P::bytes>(slot(stage, q, k), from, left > 0 ? P::bytes : 0);
            }
        } else {
            const unsigned char* start = reinterpret_cast<const unsigned char*>((uintptr_t)row & ~(uintptr_t)15);
            const int lw = lanes(c), per = lw / 4 + 1, l = c.t & (lw - 1), end = (int)((uintptr_t)row & 15) + c.D * (int)sizeof(T);
            constexpr int turns = E == 4 ? (P::count * 3 + 7) / 8 : (P::count * 9 + 31) / 32;
#pragma unroll
            for (int i = 0; i < turns; ++i) {
                const int piece = l + i * lw, k = piece / per, j = piece - k * per;
                if (k >= P::count) continue;
                const int at = 4 * (c.t - l + c.G * k) + 16 * j, left = end - at;
                fetch<16>(slot(stage, q, k) + 16 * j, left > 0 ? start + at : start, left <= 0 ? 0 : left < 16 ? left : 16);
            }
        }
    }
    // `src` and `offset` as in copy
    __device__ __forceinline__ void read(const Columns<T, E, AL>& c, int stage, int q, const void* src, long long offset, float2 (&v)[E / 2]) const {
        if constexpr (AL) {
#pragma unroll
            for (int k = 0; k < P::count; ++k) {
                uint32_t w[P::bytes / 4];
                if constexpr (P::bytes == 16) {
                    const uint4 u = *reinterpret_cast<const uint4*>(slot(stage, q, k));
                    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
                } else {
                    const uint2 u = *reinterpret_cast<const uint2*>(slot(stage, q, k));
                    w[0] = u.x, w[1] = u.y;
                }
#pragma unroll
                for (int j = 0; j < P::cols / 2; ++j) {
                    if constexpr (sizeof(T) == 4) v[k * P::cols / 2 + j] = make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
                    else v[k * P::cols / 2 + j] = pair_of_word(w[j], T());
                }
            }
        } else {
            const int off = (int)((uintptr_t)(static_cast<const T*>(src) + offset) & 15), l = 4 * (c.t & (lanes(c) - 1));
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int j = 0; j < E / 2; ++j)
                    v[j] = make_float2(*reinterpret_cast<const float*>(slot(stage, q, 2 * j) + off + l), *reinterpret_cast<const float*>(slot(stage, q, 2 * j + 1) + off + l));
            } else {
                const bool split = (off & 2) != 0;
#pragma unroll
                for (int j = 0; j < E / 2; ++j) {
                    const uint32_t* at = reinterpret_cast<const uint32_t*>(slot(stage, q, j) + (off & 12) + l);
                    uint32_t w = at[0];
                    if (split) w = __funnelshift_r(w, at[1], 16);
                    v[j] = pair_of_word(w, T());
                }
            }
        }
    }
};
__device__ __forceinline__ void ring_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int STAGES>
__device__ __forceinline__ void ring_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory"); }  // all but the newest

// The same columns straight from memory
template <typename T, int E>
__device__ __forceinline__ void load_pieces(const Columns<T, E, true>& c, const T* p, float2 (&v)[E / 2]) {
    using P = Piece<T, E, true>;
#pragma unroll
    for (int k = 0; k < P::count; ++k) {
        const int col = c.first(k);
        uint32_t w[P::bytes / 4];
        if (col < c.D) {
            if constexpr (P::bytes == 16) {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(p + col));
                w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
            } else {
                const uint2 u = __ldg(reinterpret_cast<const uint2*>(p + col));
                w[0] = u.x, w[1] = u.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < P::bytes / 4; ++j) w[j] = 0;
        }
#pragma unroll
        for (int j = 0; j < P::cols / 2; ++j) {
            if constexpr (sizeof(T) == 4) v[k * P::cols / 2 + j] = make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
            else v[k * P::cols / 2 + j] = pair_of_word(w[j], T());
        }
    }
}

template <typename T, int E, bool AL>
__device__ __forceinline__ void load_columns(const Columns<T, E, AL>& c, const void* src, long long offset, float2 (&v)[E / 2]) {
    const T* p = static_cast<const T*>(src) + offset;
#pragma unroll
    for (int j = 0; j < E / 2; ++j)
        v[j] = make_float2(c.at(2 * j) < c.D ? to_float(p[c.at(2 * j)]) : 0.f, c.at(2 * j + 1) < c.D ? to_float(p[c.at(2 * j + 1)]) : 0.f);
}

template <typename T, int E, bool AL>
__device__ __forceinline__ void store_row(const Columns<T, E, AL>& c, void* dst, long long offset, const float2 (&v)[E / 2]) {
    using P = Piece<T, E, AL>;
    T* p = static_cast<T*>(dst) + offset;
    if constexpr (AL) {
#pragma unroll
        for (int k = 0; k < P::count; ++k) {
            const int col = c.first(k);
            if (col >= c.D) continue;
            alignas(16) T e[P::cols];
#pragma unroll
            for (int j = 0; j < P::cols / 2; ++j) {
                const float2 f = v[k * P::cols / 2 + j];
                e[2 * j] = from_float<T>(f.x), e[2 * j + 1] = from_float<T>(f.y);
            }
            if constexpr (P::bytes == 16) {
                uint4 u;
                memcpy(&u, e, 16);
                __stcs(reinterpret_cast<uint4*>(p + col), u);
            } else {
                uint2 u;
                memcpy(&u, e, 8);
                __stcs(reinterpret_cast<uint2*>(p + col), u);
            }
        }
    } else {
        const bool words = sizeof(T) == 2 && ((uintptr_t)p & 2) == 0;
#pragma unroll
        for (int j = 0; j < E / 2; ++j) {
            const int a = c.at(2 * j), b = c.at(2 * j + 1);
            if (words && b < c.D) {
                const T e[2] = {from_float<T>(v[j].x), from_float<T>(v[j].y)};
                uint32_t w;
                memcpy(&w, e, 4);
                *reinterpret_cast<uint32_t*>(p + a) = w;
            } else {
                if (a < c.D) p[a] = from_float<T>(v[j].x);
                if (b < c.D) p[b] = from_float<T>(v[j].y);
            }
        }
    }
}

// The parameters of a thread's columns: its own copy in shared memory, float32, four to a 16-byte word, which only the
// thread itself reads (KEPT), or from memory at every use.
template <typename T, int E, bool AL, bool KEPT>
struct Parameters {
    const Args& p;
    float4* base;  // this thread's word of parameter 0
    int pitch;     // words of one parameter and four columns: all threads'
    static __device__ __forceinline__ void load(const Columns<T, E, AL>& c, const Args& p, int k, float2 (&v)[E / 2]) {
        const float fill = k == kGB1 || k == kGB2 ? 0.f : 1.f;
        const void* src = p.par[k];
        if (src == nullptr) {
#pragma unroll
            for (int j = 0; j < E / 2; ++j) v[j] = both(fill);
        } else if (p.pf32) {
            load_columns<float>(c, src, v);
        } else {
            if constexpr (AL)
                if (p.pvec) return load_pieces<T, E>(c, static_cast<const T*>(src), v);
            load_columns<T>(c, src, v);
        }
    }
    template <typename U>
    static __device__ __forceinline__ void load_columns(const Columns<T, E, AL>& c, const void* src, float2 (&v)[E / 2]) {
        const U* u = static_cast<const U*>(src);
#pragma unroll
        for (int j = 0; j < E / 2; ++j)
            v[j] = make_float2(c.at(2 * j) < c.D ? to_float(u[c.at(2 * j)]) : 0.f, c.at(2 * j + 1) < c.D ? to_float(u[c.at(2 * j + 1)]) : 0.f);
    }
    __device__ __forceinline__ void keep(const Columns<T, E, AL>& c, int k) const {
        if constexpr (KEPT) {
            float2 v[E / 2];
            load(c, p, k, v);
#pragma unroll
            for (int i = 0; i < E / 4; ++i) base[(k * (E / 4) + i) * pitch] = make_float4(v[2 * i].x, v[2 * i].y, v[2 * i + 1].x, v[2 * i + 1].y);
        }
    }
    __device__ __forceinline__ void read(const Columns<T, E, AL>& c, int k, float2 (&v)[E / 2]) const {
        if constexpr (KEPT) {
#pragma unroll
            for (int i = 0; i < E / 4; ++i) {
                const float4 f = base[(k * (E / 4) + i) * pitch];
                v[2 * i] = make_float2(f.x, f.y), v[2 * i + 1] = make_float2(f.z, f.w);
            }
        } else {
            load(c, p, k, v);
        }
    }
};

// Sums of N values over the threads of a row: `lanes` lanes of a warp (WARP), else the CTA. `turn` alternates between two
// sets of slots, so that one barrier per call is enough.
template <bool WARP, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int lanes, float (*slots)[2][16], int& turn) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1)
        if (!WARP || off < lanes)
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
    if constexpr (!WARP) {
        const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
        if (lane == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) slots[turn][k][wid] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            // every warp adds the warps' sums in the same order: lane w holds warp w's
            float s = lane < nw ? slots[turn][k][lane] : 0.f;
#pragma unroll
            for (int off = 8; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
            v[k] = __shfl_sync(0xffffffffu, s, 0);
        }
        turn ^= 1;
    }
}

__device__ __forceinline__ float2 sigmoid_of(float2 g) { return make_float2(sigmoid(g.x), sigmoid(g.y)); }
__device__ __forceinline__ float2 neg2(float2 v) { return make_float2(-v.x, -v.y); }

// Shape of a launch: threads of a CTA, lanes per row (rows that belong to warps), CTAs
inline int threads_of(int D) {
    if (D <= 256) return kWarpThreads;
    int G = 64;
    while (G < 512 && G * 8 < D) G *= 2;
    return G;
}
inline int lanes_of(int D) { return D <= 32 ? 8 : D <= 64 ? 16 : 32; }
inline int rows_per_cta(int D) { return D <= 256 ? kWarpThreads / lanes_of(D) : 1; }
// columns per thread, from the same bounds
inline int columns_of(int D) { return D <= 128 ? 4 : D <= 4096 ? 8 : 16; }

// whether every row of a tensor starts on a boundary of a thread's piece (null tensors do)
inline bool vec_rows(const void* ptr, long long pitch, int bytes, int elem) { return !ptr || ((uintptr_t)ptr % bytes == 0 && pitch * elem % bytes == 0); }
inline bool set_shape(Args& p, int e) {  // whether every row starts on the boundary of a thread's piece
    const int E = columns_of(p.D), bytes = E * e < 16 ? E * e : 16;
    const bool al = p.D * e % bytes == 0 && vec_rows(p.x, p.ldx, bytes, e) && vec_rows(p.gate, p.ldg, bytes, e) && vec_rows(p.res, p.ldr, bytes, e) &&
                    vec_rows(p.y, p.D, bytes, e) && vec_rows(p.res_out, p.D, bytes, e) && vec_rows(p.gy, p.ldgy, bytes, e) &&
                    vec_rows(p.gres, p.ldgr, bytes, e) && vec_rows(p.gx, p.D, bytes, e) && vec_rows(p.ggate, p.D, bytes, e) &&
                    vec_rows(p.gresid, p.D, bytes, e);
    p.pvec = al && !p.pf32;
    for (const void* q : p.par) p.pvec = p.pvec && vec_rows(q, 0, bytes, e);
    p.lanes = lanes_of(p.D);
    return al;
}
inline int check(const Args& p, int dtype, int kind, bool res) {
    if (block_elem_size(dtype) == 0 || p.M < 0 || p.D < 1 || p.act < kActNone || p.act > kActSigmoid || !(p.eps >= 0.f)) return B200_ERR_ARG;
    if (p.D > kMaxWidth) return B200_ERR_UNSUPPORTED;
    if (kind != 0 && kind != 1) return B200_ERR_ARG;
    if (kind == 0 && (p.par[kGB1] || p.par[kGB2])) return B200_ERR_ARG;
    if (p.ldx < 0 || p.ldg < 0 || p.ldr < 0 || p.ldgy < 0 || p.ldgr < 0) return B200_ERR_ARG;
    if (!res && (p.par[kGScale] || !p.par[kGW1])) return B200_ERR_ARG;
    if (p.par[kGB1] && !p.par[kGW1]) return B200_ERR_ARG;
    const int e = block_elem_size(dtype), f = p.pf32 ? 4 : e;
    if (!on_boundary(e, p.x, p.gate, p.res, p.y, p.res_out, p.gy, p.gres, p.gx, p.ggate, p.gresid)) return B200_ERR_ARG;
    for (const void* w : p.par)
        if (!on_boundary(f, w)) return B200_ERR_ARG;
    return on_boundary(16, p.stats) ? B200_OK : B200_ERR_ARG;
}

}  // namespace norm
}  // namespace b200
