// Adjoint of the block norms (the mathematics and the layout: block_norm.cuh).
//   RES:   hat2 = (res' - mean2) rstd2,  gr = gres + rstd2 (gy w2 - mean(gy w2) - hat2 mean(gy w2 hat2))
//          gw2 += gy hat2, gb2 += gy;  gresidual = gr;  gscale += gr m;  gm = scale gr
//   gate:  gn = gm act(gate),  ggate = gm n act'(gate)
//   POST:  gw1 += gn hat1, gb1 += gn;  gx = rstd1 (gn w1 - mean(gn w1) - hat1 mean(gn w1 hat1));   else gx = gn
// (without the first mean for RMS). A CTA walks over rows with a fixed stride and keeps its columns' sums in registers,
// the next two rows on their way while one is worked on.
#pragma once
#include "block_norm.cuh"

namespace b200 {
namespace norm {

// a norm's adjoint: g becomes rstd (g w - mean(g w) - hat mean(g w hat))
template <bool LAYER, bool WARP, int E>
__device__ __forceinline__ void norm_adjoint(const Args& p, float2 (&g)[E / 2], const float2 (&w)[E / 2], const float2 (&hat)[E / 2], float rstd,
                                             float (*slots)[2][16], int& turn) {
    float2 a = both(0.f), b = both(0.f);
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
        g[j] = mul2(g[j], w[j]);
        a = fma2(g[j], hat[j], a);
        if (LAYER) b = add2(g[j], b);
    }
    const float inv = 1.f / (float)p.D;
    if constexpr (LAYER) {
        float s[2] = {a.x + a.y, b.x + b.y};
        row_sum<WARP, 2>(s, p.lanes, slots, turn);
#pragma unroll
        for (int j = 0; j < E / 2; ++j) g[j] = mul2(fma2(hat[j], both(-s[0] * inv), add2(g[j], both(-s[1] * inv))), both(rstd));
    } else {
        float s[1] = {a.x + a.y};
        row_sum<WARP, 1>(s, p.lanes, slots, turn);
#pragma unroll
        for (int j = 0; j < E / 2; ++j) g[j] = mul2(fma2(hat[j], both(-s[0] * inv), g[j]), both(rstd));
    }
}

template <typename T, bool LAYER, bool POST, bool RES, bool WARP, int E, bool AL>
__global__ void __launch_bounds__(WARP ? kWarpThreads : 512, WARP ? 4 : 1) norm_bwd_kernel(const Args p) {
    using K = Keeps<T, LAYER, RES, WARP, E, AL, true>;
    constexpr int N = K::tensors, SUMS = K::params, STAGES = K::stages, H = E / 2;  // x, gate, gy, residual, gres
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float slots[2][2][16];
    int turn = 0;
    const int threads = blockDim.x;
    Columns<T, E, AL> c;
    c.t = WARP ? threadIdx.x & (p.lanes - 1) : threadIdx.x, c.G = WARP ? p.lanes : threads, c.D = p.D;
    const Parameters<T, E, AL, K::kept> par = {p, reinterpret_cast<float4*>(smem) + threadIdx.x, threads};
    unsigned char* ring_at = smem + (K::kept ? K::par * threads : 0);
    const auto ring = Ring<T, E, AL, N>::at(c, ring_at);
    if constexpr (POST) par.keep(c, kGW1);
    if constexpr (POST && LAYER) par.keep(c, kGB1);
    if constexpr (RES) par.keep(c, kGW2), par.keep(c, kGScale);
    const int per = WARP ? threads / p.lanes : 1;
    const long long stride = (long long)gridDim.x * per, mine = WARP ? threadIdx.x / p.lanes : 0;
    const bool gated = p.gate != nullptr, silu = p.act == kActSilu;
    auto request = [&](long long row, int stage) {
        if (STAGES > 0 && row < p.M) {
            ring.copy(c, stage, 0, p.x, row * p.ldx);
            if (gated) ring.copy(c, stage, 1, p.gate, row * p.ldg);
            ring.copy(c, stage, 2, p.gy, row * p.ldgy);
            if constexpr (RES) {
                ring.copy(c, stage, 3, p.res, row * p.ldr);
                if (p.gres != nullptr) ring.copy(c, stage, 4, p.gres, row * p.ldgr);
            }
        }
        ring_commit();
    };
    float2 acc[SUMS][H];
#pragma unroll
    for (int s = 0; s < SUMS; ++s)
#pragma unroll
        for (int j = 0; j < H; ++j) acc[s][j] = both(0.f);
    long long base = (long long)blockIdx.x * per;
    for (int s = 0; s < STAGES - 1; ++s) request(base + s * stride + mine, s);
    int stage = 0;
    float4 st_next = base + mine < p.M ? *reinterpret_cast<const float4*>(p.stats + 4 * (base + mine)) : make_float4(0.f, 0.f, 0.f, 0.f);
    for (; base < p.M; base += stride) {
        const long long row = base + mine;
        const bool live = row < p.M;
        const float4 st = st_next;
        if (row + stride < p.M) st_next = *reinterpret_cast<const float4*>(p.stats + 4 * (row + stride));
        if constexpr (STAGES > 0) {
            ring.together();
            request(row + (STAGES - 1) * stride, stage == 0 ? STAGES - 1 : stage - 1);
            ring_wait<STAGES>();
            ring.together();
        }
        auto read = [&](int q, const void* src, long long pitch, float2(&v)[H]) {
            if (!live) {
#pragma unroll
                for (int j = 0; j < H; ++j) v[j] = both(0.f);
            } else if constexpr (STAGES > 0) {
                ring.read(c, stage, q, src, row * pitch, v);
            } else if constexpr (AL) {
                load_pieces<T, E>(c, static_cast<const T*>(src) + row * pitch, v);
            } else {
                load_columns<T, E, AL>(c, src, row * pitch, v);
            }
        };
        // n = w1 hat1 + b1 (or x), the gate's sigmoid (without SiLU: it minus one) and value, m = n value
        float2 hat1[H], n[H], sig[H], val[H], gm[H], v[H];
        read(0, p.x, p.ldx, n);
        if constexpr (POST) {
            par.read(c, kGW1, v);
#pragma unroll
            for (int j = 0; j < H; ++j) {
                hat1[j] = LAYER ? mul2(mul2(add2(n[j], both(-st.x)), both(st.y)), c.inside(j)) : mul2(n[j], both(st.y));
                n[j] = mul2(hat1[j], v[j]);
            }
            if constexpr (LAYER) {
                par.read(c, kGB1, v);
#pragma unroll
                for (int j = 0; j < H; ++j) n[j] = add2(n[j], v[j]);
            }
        }
        if (gated) {
            read(1, p.gate, p.ldg, v);
#pragma unroll
            for (int j = 0; j < H; ++j) {
                sig[j] = sigmoid_of(v[j]);
                val[j] = silu ? mul2(sig[j], v[j]) : sig[j];
                // the slope s (1 - s) of an open gate: 1 - s is the function of -v, the difference keeps nothing of it
                if (!silu) sig[j] = neg2(sigmoid_of(neg2(v[j])));
            }
        } else {
#pragma unroll
            for (int j = 0; j < H; ++j) val[j] = both(1.f);
        }
        read(2, p.gy, p.ldgy, gm);
        if constexpr (RES) {
            float2 hat2[H];
            read(3, p.res, p.ldr, hat2);
            par.read(c, kGScale, v);
#pragma unroll
            for (int j = 0; j < H; ++j) {
                const float2 r = fma2(v[j], mul2(n[j], val[j]), hat2[j]);
                hat2[j] = LAYER ? mul2(mul2(add2(r, both(-st.z)), both(st.w)), c.inside(j)) : mul2(r, both(st.w));
                acc[kGW2][j] = fma2(gm[j], hat2[j], acc[kGW2][j]);
                if constexpr (LAYER) acc[kGB2][j] = add2(gm[j], acc[kGB2][j]);
            }
            par.read(c, kGW2, v);
            norm_adjoint<LAYER, WARP, E>(p, gm, v, hat2, st.w, slots, turn);
            if (p.gres != nullptr) {
                read(4, p.gres, p.ldgr, v);
#pragma unroll
                for (int j = 0; j < H; ++j) gm[j] = add2(gm[j], v[j]);
            }
            if (live) store_row<T, E, AL>(c, p.gresid, row * p.D, gm);
            par.read(c, kGScale, v);
#pragma unroll
            for (int j = 0; j < H; ++j) {
                // (columns past the width hold zeros in n and val's product, or in gm)
                acc[kGScale][j] = fma2(gm[j], mul2(n[j], val[j]), acc[kGScale][j]);
                gm[j] = mul2(gm[j], v[j]);
            }
        }
        if (gated) {
#pragma unroll
            for (int j = 0; j < H; ++j) {
                // SiLU: g s (1 - s) + s; the logistic function: s (1 - s), with s - 1 in `sig`
                const float2 slope = fma2(neg2(val[j]), sig[j], silu ? add2(val[j], sig[j]) : both(0.f));
                n[j] = mul2(mul2(gm[j], n[j]), slope);
                gm[j] = mul2(gm[j], val[j]);
            }
            if (live && p.ggate != nullptr) store_row<T, E, AL>(c, p.ggate, row * p.D, n);
        }
        if constexpr (POST) {
            par.read(c, kGW1, v);
#pragma unroll
            for (int j = 0; j < H; ++j) {
                acc[kGW1][j] = fma2(gm[j], hat1[j], acc[kGW1][j]);
                if constexpr (LAYER) acc[kGB1][j] = add2(gm[j], acc[kGB1][j]);
            }
            norm_adjoint<LAYER, WARP, E>(p, gm, v, hat1, st.y, slots, turn);
        }
        if (live && p.gx != nullptr) store_row<T, E, AL>(c, p.gx, row * p.D, gm);
        stage = stage + 1 >= STAGES ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // one partial row per CTA and sum
#pragma unroll
    for (int s = 0; s < SUMS; ++s) {
        const bool kept = s == kGW1 || s == kGB1 ? POST : RES;
        if (!kept) continue;
        float* out = p.part + ((long long)blockIdx.x * SUMS + s) * p.D;
        if constexpr (WARP) {
            float2* red = reinterpret_cast<float2*>(smem);  // [pairs][threads]
            __syncthreads();
#pragma unroll
            for (int j = 0; j < H; ++j) red[j * threads + threadIdx.x] = acc[s][j];
            __syncthreads();
            if (threadIdx.x < p.lanes) {
#pragma unroll
                for (int j = 0; j < H; ++j) {
                    float2 t = both(0.f);
                    for (int r = 0; r < per; ++r) t = add2(t, red[j * threads + r * p.lanes + threadIdx.x]);
                    if (c.at(2 * j) < c.D) out[c.at(2 * j)] = t.x;
                    if (c.at(2 * j + 1) < c.D) out[c.at(2 * j + 1)] = t.y;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < H; ++j) {
                if (c.at(2 * j) < c.D) out[c.at(2 * j)] = acc[s][j].x;
                if (c.at(2 * j + 1) < c.D) out[c.at(2 * j + 1)] = acc[s][j].y;
            }
        }
    }
}

struct Sums {
    void* out[5];
    int f32;
};
// out[s][d] = sum over CTAs of part[CTA][s][d], in a fixed order: 32 columns per block, 32 threads per column
template <typename T>
__global__ void __launch_bounds__(1024) norm_columns_kernel(const float* __restrict__ part, int rows, int sums, int D, const Sums o) {
    __shared__ float red[32][33];
    const int s = blockIdx.y, dl = threadIdx.x & 31, k = threadIdx.x >> 5, d = blockIdx.x * 32 + dl;
    if (o.out[s] == nullptr) return;
    float t = 0.f;
    if (d < D)
        for (int r = k; r < rows; r += 32) t += part[((long long)r * sums + s) * D + d];
    red[k][dl] = t;
    __syncthreads();
    if (k == 0 && d < D) {
        t = 0.f;
        for (int j = 0; j < 32; ++j) t += red[j][dl];
        if (o.f32) static_cast<float*>(o.out[s])[d] = t;
        else static_cast<T*>(o.out[s])[d] = from_float<T>(t);
    }
}

// CTAs of the adjoint: 512 threads per SM, no more than there are rows to share
inline long long grid_of(long long M, int D) {
    const long long rows = (M + rows_per_cta(D) - 1) / rows_per_cta(D), most = 148LL * (512 / threads_of(D));
    return rows < most ? rows : most;
}

template <typename T, bool LAYER, bool POST, bool RES, bool WARP, int E, bool AL>
int launch_bwd_as(const Args& p, int grid, cudaStream_t st) {
    const int threads = threads_of(p.D);
    size_t smem = (size_t)threads * Keeps<T, LAYER, RES, WARP, E, AL, true>::bytes;
    if (WARP && smem < (size_t)threads * E * 4) smem = (size_t)threads * E * 4;  // the sums of a CTA's rows meet there
    const auto kernel = norm_bwd_kernel<T, LAYER, POST, RES, WARP, E, AL>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return B200_ERR_LAUNCH;
    kernel<<<grid, threads, smem, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_LAUNCH;
}
template <typename T, bool LAYER, bool POST, bool RES, bool AL>
int launch_bwd(const Args& p, const Sums& o, cudaStream_t st) {
    const int grid = (int)grid_of(p.M, p.D);
    if (grid > 0) {
        const int rc = p.D <= 128    ? launch_bwd_as<T, LAYER, POST, RES, true, 4, AL>(p, grid, st)
                       : p.D <= 256  ? launch_bwd_as<T, LAYER, POST, RES, true, 8, AL>(p, grid, st)
                       : p.D <= 4096 ? launch_bwd_as<T, LAYER, POST, RES, false, 8, AL>(p, grid, st)
                                     : launch_bwd_as<T, LAYER, POST, RES, false, 16, AL>(p, grid, st);
        if (rc != B200_OK) return rc;
    }
    constexpr int sums = LAYER ? 5 : 3;
    norm_columns_kernel<T><<<dim3((p.D + 31) / 32, sums), 1024, 0, st>>>(p.part, grid, sums, p.D, o);
    return cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_LAUNCH;
}
template <typename T, bool AL>
int pick_bwd(const Args& p, const Sums& o, bool layer, bool post, bool res, cudaStream_t st) {
    if (layer)
        return !res ? launch_bwd<T, true, true, false, AL>(p, o, st) : post ? launch_bwd<T, true, true, true, AL>(p, o, st) : launch_bwd<T, true, false, true, AL>(p, o, st);
    return !res ? launch_bwd<T, false, true, false, AL>(p, o, st) : post ? launch_bwd<T, false, true, true, AL>(p, o, st) : launch_bwd<T, false, false, true, AL>(p, o, st);
}

template <bool AL>
int bwd_of(const Args& p, const Sums& o, int dtype, bool layer, bool post, bool res, cudaStream_t st) {
    if (dtype == B200_F32) return pick_bwd<float, AL>(p, o, layer, post, res, st);
    if (dtype == B200_BF16) return pick_bwd<__nv_bfloat16, AL>(p, o, layer, post, res, st);
    return pick_bwd<__half, AL>(p, o, layer, post, res, st);
}
// the kernels for rows on and off 16-byte boundaries, each in a unit of its own: they take minutes to compile
int bwd_aligned(const Args& p, const Sums& o, int dtype, bool layer, bool post, bool res, cudaStream_t st);
int bwd_unaligned(const Args& p, const Sums& o, int dtype, bool layer, bool post, bool res, cudaStream_t st);

}  // namespace norm
}  // namespace b200
