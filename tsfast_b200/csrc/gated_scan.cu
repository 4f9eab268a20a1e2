// Gated linear recurrence with its gates fused in (float32, bfloat16 or float16 sequences, float32 state):
//   rho = sigmoid(r_t), iota = sigmoid(i_t), l = -c softplus(lam) rho, a_t = e^l, beta_t = sqrt(1 - e^{2l}),
//   h_t = a_t h_{t-1} + beta_t iota x_t
// per channel, over a batch [B, L, D] or over sequences packed end to end [T, D]; its adjoint
//   g~_t = gh_t + a_{t+1} g~_{t+1},   gx = g~ beta iota,   gi = gx x (1 - iota),
//   w = l (a g~ h_{t-1} - (a^2 / beta) g~ iota x),   gr = w (1 - rho),   glam = sigmoid(lam)/softplus(lam) sum_t w
// (w is the gradient of l times l: both l's derivatives, by r and by lam, are l times something, and l / beta stays
// finite where beta goes to zero); and the form for one token per row against a cache of states.
//
// Numerics: u = e^l - 1 and a are both computed to full relative accuracy (to base 2: the integer part goes to the exponent, the rest
// through a polynomial fitted to the smallest largest relative error by Lawson's iteration), so a and beta^2 = -u (2 + u) are
// right where a is close to 1, which is where such a layer works, and where it is small. The state, the gates, all products and all
// sums are float32; sequences are rounded once, when they are stored. The adjoint recomputes the states from
// float32 states kept at every tile instead of reading the rounded h back: one tensor less to read, and no error
// of 2^-9 in h_{t-1}.
//
// Layout of the work: a chain is (sequence, 256 bytes of channels). A CTA takes tiles of consecutive steps of a chain; a lane
// has two or four neighbouring channels, each of seven warps a segment of four steps held in registers, so a warp reads and writes 256-byte
// pieces of rows. A warp fetches its own rows (cp.async, a private ring) and needs nobody else's.
// A segment is an affine map of the state that enters it. The seven maps go through shared memory to an eighth warp, which
// folds them from the carry and hands every warp the state that enters its segment; the warps meanwhile compute the
// gates of the next tile, so no warp waits for another between two tiles (one barrier per exchange with all eight warps
// folding took 178 us for 8 x 4096 x 2048 bf16, of which 128 remained without any arithmetic).
// Where there are few chains (one long prompt), a cluster of C CTAs takes C consecutive tiles of the same chain at a
// time, and the folding warps pass the tiles' maps through distributed shared memory with st.async: no flags in global
// memory, nothing to reset, a fixed order of every sum. All waits are bounded (b200_block_status reads the error word).
//
// Measured (bytes are the tensors once: 4 forward, 7 in the adjoint): 8 x 4096 x 2048 float32 217 us and 362 us, 4.9 and 5.2
// TB/s, near what memory gives; bfloat16 153 and 332 us, 3.5 and 2.8 TB/s. In 16 bits it is the arithmetic that bounds them, not
// memory: 39 and 74 instructions per channel and step, issued in 0.51 and 0.45 of the cycles by the sixteen warps that the
// registers allow, the rest being latencies of the chain loads - gates - maps - states. A deeper ring does not help (adjoint:
// 311 us with three stages and one copy of the maps, 307 with two; forward: 160 us with four stages, 156 with three). Decays below
// 2^-1/2 take the longer form of the exponential: 173 and 354 us. The adjoint's 1 - rho and 1 - iota cost it a second exponential
// each, and a reciprocal (312 us with the differences, which lose their digits at open gates).
// One 65536 x 1024 prompt (bfloat16, clusters of twelve): 226 us forward.
#include "block.cuh"

namespace b200 {
namespace gated {

constexpr int kWarps = 7, kThreads = (kWarps + 1) * 32;  // eight warps with the one that folds: 128 registers at two CTAs per SM
constexpr int kSteps = 4, kTile = kSteps * kWarps;       // steps of a segment and of a tile
constexpr int kMaxCluster = 12;                           // above 8 a cluster needs the device's consent (it has it)

// Channels of a chain: 128 in 16 bits (two pairs per lane), 64 in float32, or 64 in 16 bits where chains are few.
template <int NP>
struct Lanes {
    static constexpr int chans = 64 * NP, per_lane = 2 * NP;
};
template <bool BWD>
struct Shape {
    static constexpr int tensors = BWD ? 4 : 3;
    static constexpr int stages = BWD ? 2 : 3;  // of a warp's ring; a third one leaves the adjoint one CTA per SM: 441 us against 307
};

__device__ __forceinline__ float2 unpack(uint32_t v, __nv_bfloat16) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack(uint32_t v, __half) {
    __half2 h;
    memcpy(&h, &v, 4);
    return __half22float2(h);
}

// two neighbouring channels from memory that is aligned to the pair
template <typename T>
__device__ __forceinline__ float2 load2(const void* p) {
    if constexpr (sizeof(T) == 4) return *static_cast<const float2*>(p);
    else return unpack(*static_cast<const uint32_t*>(p), T());
}
// a lane's channels: in one go, or the first n of them one by one
template <typename T, int NP>
__device__ __forceinline__ void store_lane(T* p, const Pair (&v)[NP], bool whole, int n) {
    constexpr int V = 2 * NP;
    T o[V];
#pragma unroll
    for (int k = 0; k < NP; ++k) o[2 * k] = from_float<T>(pair2(v[k]).x), o[2 * k + 1] = from_float<T>(pair2(v[k]).y);
    if (whole) {
        if (n > 0) {
            if constexpr (V * sizeof(T) == 8) {
                uint2 w;
                memcpy(&w, o, 8);
                __stcs(reinterpret_cast<uint2*>(p), w);
            } else {
                uint32_t w;
                memcpy(&w, o, 4);
                __stcs(reinterpret_cast<unsigned int*>(p), w);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < n) p[e] = o[e];
    }
}
// float32 rows of the states' arrays
template <int NP>
__device__ __forceinline__ void load_state(const float* p, int n, Pair (&v)[NP]) {
#pragma unroll
    for (int k = 0; k < NP; ++k) v[k] = bits2(make_float2(2 * k < n ? p[2 * k] : 0.f, 2 * k + 1 < n ? p[2 * k + 1] : 0.f));
}
template <int NP>
__device__ __forceinline__ void store_state(float* p, int n, const Pair (&v)[NP]) {
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        if (2 * k < n) p[2 * k] = pair2(v[k]).x;
        if (2 * k + 1 < n) p[2 * k + 1] = pair2(v[k]).y;
    }
}

// The larger of two, NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The constants of the functions below, in both halves of a register pair
struct Constants {
    Pair nlog2e, one, neg1, c[6];
};
__device__ __forceinline__ Constants constants() {
    Constants k;
    k.nlog2e = resident(-1.4426950408889634f), k.one = resident(1.f), k.neg1 = resident(-1.f);
    k.c[0] = resident(0x1.62e43p-1f), k.c[1] = resident(0x1.ebfbdep-3f), k.c[2] = resident(0x1.c6af6ep-5f);
    k.c[3] = resident(0x1.3b2bap-7f), k.c[4] = resident(0x1.5f0816p-10f), k.c[5] = resident(0x1.4308fap-13f);
    return k;
}
// sigmoid of two values. (The reciprocal by Newton's iteration on the multiply-add pipe instead costs nine instructions more
// per pair and 7 % of the forward pass: issue slots are shorter than the special-function unit.)
__device__ __forceinline__ Pair sigmoid2(const Constants& k, Pair x) {
    const float2 t = pair2(mul2(x, k.nlog2e));
    const float2 d = pair2(add2(bits2(make_float2(ex2(t.x), ex2(t.y))), k.one));
    return bits2(make_float2(rcp(d.x), rcp(d.y)));
}
// 1 - s of s = sigmoid(x), as e^-x s: the difference keeps nothing of it where the gate is open (at x = 10 it is 4.5e-5, and s is
// known to 2^-24). The limit keeps infinity times zero away where s has gone to zero.
__device__ __forceinline__ Pair complement2(const Constants& k, Pair x, Pair s) {
    const float2 t = pair2(mul2(x, k.nlog2e));
    return mul2(bits2(make_float2(ex2(fminf(t.x, 126.f)), ex2(fminf(t.y, 126.f)))), s);
}
// The same where s is not at hand, as the function of -x
__device__ __forceinline__ Pair co_sigmoid2(const Constants& k, Pair x) {
    const float2 t = pair2(mul2(x, k.nlog2e));
    const float2 d = pair2(add2(bits2(make_float2(ex2(-t.x), ex2(-t.y))), k.one));
    return bits2(make_float2(rcp(d.x), rcp(d.y)));
}
// Of two l <= 0: u = 2^l - 1 and a = 2^l, each to the last bits (a - 1 keeps nothing of u where a is close to one, and u + 1
// nothing of a where a is small). SLOW: l >= -1/2 is known, and the polynomial is all it takes. Else its integer part
// goes to the exponent; a below 2^-126 is given as 2^-126. A NaN passes through.
struct Decay {
    Pair u, a;
};
template <bool SLOW>
__device__ __forceinline__ Decay decay2(const Constants& k, Pair l2) {
    Pair f = l2, s = 0;
    if constexpr (!SLOW) {
        const float2 c = pair2(l2);
        l2 = bits2(make_float2(max_nan(c.x, -126.f), max_nan(c.y, -126.f)));
        const Pair t = add2(l2, bits2(both(12582912.f)));  // 1.5 * 2^23 + l: the low bits hold round(l)
        f = fma2(add2(t, bits2(both(-12582912.f))), k.neg1, l2);
        const float2 i = pair2(t);
        s = bits2(make_float2(__int_as_float(__float_as_int(i.x) * (1 << 23) + 0x3f800000), __int_as_float(__float_as_int(i.y) * (1 << 23) + 0x3f800000)));
    }
    Pair q = fma2(k.c[5], f, k.c[4]);
    q = fma2(q, f, k.c[3]);
    q = fma2(q, f, k.c[2]);
    q = fma2(q, f, k.c[1]);
    q = fma2(q, f, k.c[0]);
    q = mul2(f, q);
    if constexpr (SLOW) return {q, add2(q, k.one)};
    else return {fma2(s, q, add2(s, k.neg1)), fma2(s, q, s)};
}
// u = a - 1: -beta^2 = u (2 + u)
__device__ __forceinline__ Pair minus_beta2(Pair u) { return fma2(u, u, add2(u, u)); }
// Whether exp(-c softplus(lam)) >= 2^-1/2 for all channels of a warp: then so is every decay, whatever its gate. Layers
// that remember start there (0.9 and above); the short form saves nine instructions per pair.
template <int NP>
__device__ __forceinline__ bool slow_decays(const Pair (&nsp2)[NP]) {
    bool slow = true;
#pragma unroll
    for (int e = 0; e < NP; ++e) slow = slow && pair2(nsp2[e]).x >= -0.5f && pair2(nsp2[e]).y >= -0.5f;
    return __all_sync(0xffffffffu, slow);
}
__device__ __forceinline__ float root(float x) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

// -c softplus(lam) of a lane's channels (zero past the width)
template <int NP>
__device__ __forceinline__ void decay_rates(const float* lam, float c, int n, Pair (&v)[NP]) {
    load_state<NP>(lam, n, v);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        const float2 l = pair2(v[k]);
        v[k] = bits2(make_float2(2 * k < n ? -c * softplus(l.x) : 0.f, 2 * k + 1 < n ? -c * softplus(l.y) : 0.f));
    }
}

struct Seq {  // one operand: pointer, element strides of the batch row and of the token
    const void* p;
    long long sb, st;
};
struct Args {
    Seq in[4];          // x, r, i, gh
    void* out[3];       // forward: h; adjoint: gx, gr, gi (dense rows of D)
    const float* lam;
    const float* h0;    // [S, D] or null
    float* hlast;       // forward: final state; adjoint: gradient of h0 (null: not wanted)
    const float* glast; // adjoint: gradient of the final state or null
    float* chk;         // state entering every tile, [slots, D] (forward: null = not kept)
    float* part;        // adjoint: sums of w, one row per CTA of a chain, [S * C, D]
    const void* cu;     // boundaries of packed sequences (int32 or int64) or null
    int cu64;
    long long S, L, T;  // sequences, steps of each (batch), rows of the buffer (packed)
    int D;
    int ctiles, C;
    float c;
    int whole;          // outputs: rows of whole lanes of channels on an aligned base
    int until;          // forward: the step with which the first CTA of every chain falls silent (the probe's; else past the last)
};

__device__ __forceinline__ long long boundary(const Args& p, long long k) {
    long long v = p.cu64 ? static_cast<const long long*>(p.cu)[k] : (long long)static_cast<const int*>(p.cu)[k];
    return v < 0 ? 0 : v > p.T ? p.T : v;
}

// where a chain's rows are: offset of its first row in the outputs, first row for the inputs, length, first tile's slot
struct Chain {
    long long row0, slot0;
    int len;
    long long b;  // batch row of the inputs (0 when packed)
    long long t0; // first token of the inputs inside the batch row
};
__device__ __forceinline__ Chain locate(const Args& p, long long seq) {
    Chain c;
    if (p.cu == nullptr) {
        c.b = seq, c.t0 = 0, c.row0 = seq * p.L, c.len = (int)p.L;
        c.slot0 = seq * ((p.L + kTile - 1) / kTile);
    } else {
        const long long s = boundary(p, seq), e = boundary(p, seq + 1);
        c.b = 0, c.t0 = s, c.row0 = s, c.len = e > s ? (int)(e - s) : 0;
        c.slot0 = s / kTile + seq;  // a sequence that ends in row e uses slots below e / kTile + seq + 1
    }
    return c;
}

// ------------------------------------------------------------------------------------------- a warp's rows in shared memory
// A row of a segment is 128 or 256 bytes. MIS: the rows do not start on 16-byte boundaries (an odd width, a slice at an odd
// place): whole 16-byte granules are fetched, one more per row, and a row is read at its own offset. A granule is
// fetched only if a wanted byte lies in it, and not past the row's last channel.
template <typename T, bool MIS, int NP, bool BWD>
struct Rows {
    static constexpr int pitch = Lanes<NP>::chans * (int)sizeof(T) + (MIS ? 16 : 0);
    static constexpr int granules = pitch / 16;
    static constexpr int bytes = kSteps * pitch;
    static constexpr int stage = Shape<BWD>::tensors * bytes;
    static constexpr int ring = Shape<BWD>::stages * stage;  // of one warp
};

__device__ __forceinline__ void cp16(uint32_t dst, const unsigned char* src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
// Rows `row0` .. of every operand (at most `valid` of them) into one of the warp's stages. What lies past the last row or
// channel is left as it was: the readers know how many steps there are, and channels past the width are not stored.
template <typename T, bool MIS, int NP, bool BWD, int N>
__device__ __forceinline__ void fetch(uint32_t stage, const unsigned char* const (&src)[N], const long long (&step)[N], int row0, int valid,
                                      int row_bytes) {
    using R = Rows<T, MIS, NP, BWD>;
    const int lane = threadIdx.x & 31;
    if constexpr (!MIS) {
        constexpr int per_pass = 32 / R::granules;  // a lane has one granule of every per_pass-th row
        const int row = lane / R::granules, k = lane % R::granules;
        const int n = min(row_bytes - 16 * k, 16);
        if (n <= 0) return;
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const unsigned char* g = src[q] + (row0 + row) * step[q] + 16 * k;
#pragma unroll
            for (int i = 0; i < kSteps / per_pass; ++i) {
                if (row + i * per_pass < valid) cp16(stage + q * R::bytes + i * per_pass * R::pitch + lane * 16, g, n);
                g += per_pass * step[q];
            }
        }
    } else {
#pragma unroll
        for (int q = 0; q < N; ++q) {
#pragma unroll
            for (int c0 = 0; c0 < kSteps * R::granules; c0 += 32) {
                const int c = c0 + lane, row = c / R::granules, k = c - row * R::granules;
                if (c >= kSteps * R::granules || row >= valid) continue;
                const unsigned char* first = src[q] + (row0 + row) * step[q];
                const unsigned char* g = reinterpret_cast<const unsigned char*>(reinterpret_cast<uintptr_t>(first) & ~(uintptr_t)15) + 16 * k;
                const long long n = first + row_bytes - g;
                if (n > 0) cp16(stage + q * R::bytes + row * R::pitch + k * 16, g, n > 16 ? 16 : (int)n);
            }
        }
    }
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// the lane's channels of one row; `first` is the row's address in global memory (its offset within 16 bytes counts)
template <typename T, bool MIS, int NP>
__device__ __forceinline__ void row_lane(const unsigned char* row, int lane, uint32_t first, Pair (&v)[NP]) {
    const unsigned char* p = row + lane * (2 * NP * (int)sizeof(T));
    if constexpr (!MIS) {
        if constexpr (NP == 1) {
            v[0] = bits2(load2<T>(p));
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(p);
            v[0] = bits2(unpack(w.x, T())), v[1] = bits2(unpack(w.y, T()));
        }
    } else {
        const T* e = reinterpret_cast<const T*>(p + (first & 15u));
#pragma unroll
        for (int k = 0; k < NP; ++k) v[k] = bits2(make_float2(to_float(e[2 * k]), to_float(e[2 * k + 1])));
    }
}

template <bool V>
struct Bool {
    static constexpr bool value = V;
};

// An affine map of a pair of channels' states: decays and sums. Applied to a state, and put after another map
struct alignas(16) Map {
    Pair decay, sum;
};
__device__ __forceinline__ Pair apply(const Map& m, Pair h) { return fma2(m.decay, h, m.sum); }
__device__ __forceinline__ Map after(const Map& m, const Map& first) { return {mul2(m.decay, first.decay), apply(m, first.sum)}; }

// ------------------------------------------------------------------------------------------- clusters
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Maps travel with st.async, which signals the receiver's mbarrier by bytes: no fence and no cluster barrier per tile
// (the barrier's release waits for the tile's global stores too: 20 % of the forward pass).
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void put_remote(const Map* local, uint64_t* bar, int rank, const Map& v) {
    uint32_t a, b;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(smem_u32(bar)), "r"(rank));
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];" ::"r"(a), "l"(v.decay), "l"(v.sum), "r"(b)
                 : "memory");
}
__device__ __forceinline__ void expect(uint64_t* bar, int bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Bounded wait (a poll waits 4 us itself). One that runs out is remembered in `lost`: later waits return at once, the results are
// wrong, and the error word says so.
constexpr int kWaitLimit = 1 << 18;  // polls: about a second
__device__ __forceinline__ void await(uint64_t* bar, uint32_t parity, bool& lost) {
    for (int i = 0; i < kWaitLimit && !lost; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return;
    }
    lost = true;
}

// What the warps of a CTA, and the CTAs of a cluster, tell one another; two of each, for alternating tiles.
struct Barriers {
    uint64_t maps[2];   // the seven warps' maps are written
    uint64_t start[2];  // the states that enter the segments are written
    uint64_t peers[2];  // the tiles' maps of all CTAs have come in
};
__device__ __forceinline__ void open_exchange(int C, Barriers& b) {
    if (threadIdx.x == 0) {
        for (int k = 0; k < 2; ++k) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&b.maps[k])), "r"(kWarps) : "memory");
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&b.start[k])) : "memory");
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&b.peers[k])) : "memory");
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (C > 1) cluster_sync();  // every CTA of the cluster is there before anything is written into it
    else __syncthreads();
}
__device__ unsigned int exchange_lost;  // B200_ERR_TIMEOUT once a wait ran out
__device__ __forceinline__ void close_exchange(int C, bool lost) {
    if (lost) atomicExch(&exchange_lost, (unsigned int)B200_ERR_TIMEOUT);
    if (C > 1) {
        cluster_sync();  // nobody leaves while a map may be on its way to it: all have been sent, and who has not lost a wait has them all
        if (__syncthreads_or(lost))
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // who has lost one gives the rest a bounded time to land
    } else {
        __syncthreads();
    }
}
// The folding warp of every CTA tells all CTAs of its cluster its tile's maps, and folds theirs from the carry: the states
// that enter this CTA's tile (in `enter`); the carry becomes those behind the last CTA's.
// A lane that has lost a wait sends and expects nothing any more (`to` becomes zero; it is C before): the barrier would be
// arrived at twice in one phase. So all CTAs lose theirs.
template <int NP>
__device__ __forceinline__ void exchange(Map (*peers)[NP][32], Barriers& b, int C, int rank, int s, const Map (&mine)[NP], Pair (&enter)[NP],
                                         Pair (&carry)[NP], int& to, bool& lost) {
    const int buf = s & 1, lane = threadIdx.x & 31;
    if (lane == 0 && to > 0) expect(&b.peers[buf], C * 32 * NP * (int)sizeof(Map));
    for (int c = 0; c < to; ++c)
#pragma unroll
        for (int k = 0; k < NP; ++k) put_remote(&peers[buf * C + rank][k][lane], &b.peers[buf], c, mine[k]);
    await(&b.peers[buf], (uint32_t)(s >> 1) & 1u, lost);
    if (lost) to = 0;
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            if (c == rank) enter[k] = carry[k];
            carry[k] = apply(peers[buf * C + c][k][lane], carry[k]);
        }
}

// zeros in the rows that belong to no sequence: before the first boundary and behind the last
template <typename T, int NP>
__device__ void clear_spare_rows(const Args& p, int n_out, int ct, int rank) {
    const long long head = boundary(p, 0), tail = boundary(p, p.S);
    const int lane = threadIdx.x & 31, d = ct * Lanes<NP>::chans + 2 * NP * lane;
    const Pair zeros[NP] = {};
    const long long stride = (long long)p.C * (kThreads / 32);
    for (long long t = (long long)rank * (kThreads / 32) + (threadIdx.x >> 5); t < p.T; t += stride) {
        if (t >= head && t < tail) {  // on to the rows behind the last sequence, in this thread's stride
            t += (tail - t + stride - 1) / stride * stride;
            if (t >= p.T) break;
        }
        for (int o = 0; o < n_out; ++o) store_lane<T, NP>(static_cast<T*>(p.out[o]) + t * p.D + d, zeros, p.whole, p.D - d);
    }
}

// ------------------------------------------------------------------------------------------- forward
template <typename T, bool MIS, int NP>
__global__ void __launch_bounds__(kThreads, 2) gated_fwd_kernel(const Args p) {
    using R = Rows<T, MIS, NP, false>;
    constexpr int ST = Shape<false>::stages, TS = kSteps;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ Map maps[2][kWarps][NP][32];
    __shared__ Pair start[2][kWarps][NP][32];  // the states that enter a segment
    Map(*const peers)[NP][32] = reinterpret_cast<Map(*)[NP][32]>(smem + kWarps * R::ring);  // [2 * C], in clusters only
    __shared__ __align__(8) Barriers bars;
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int C = p.C, rank = (int)(blockIdx.x % C);
    const long long chain = blockIdx.x / C;
    const int ct = (int)(chain % p.ctiles);
    const long long seq = chain / p.ctiles;
    if (seq == p.S) {  // (packed only) every CTA of a cluster takes this way together
        clear_spare_rows<T, NP>(p, 1, ct, rank);
        return;
    }
    const Chain ch = locate(p, seq);
    const int d = ct * Lanes<NP>::chans + 2 * NP * lane, n = p.D - d;  // the lane's first channel, and how many there are from it on
    const int tiles = (ch.len + kTile - 1) / kTile, steps = (tiles + C - 1) / C;
    bool lost = false;
    open_exchange(C, bars);

    if (wid == kWarps) {
        // ---------------------------------------------------------------- the warp that folds
        int to = C;
        Pair carry[NP] = {}, h[NP];
        if (p.h0 != nullptr) load_state<NP>(p.h0 + seq * p.D + d, n, carry);
        const int mine = rank == 0 ? min(steps, p.until) : steps;
        for (int s = 0; s < mine; ++s) {
            const int buf = s & 1, tile = s * C + rank;
            await(&bars.maps[buf], (uint32_t)(s >> 1) & 1u, lost);
            if (C == 1) {
#pragma unroll
                for (int k = 0; k < NP; ++k) h[k] = carry[k];
            } else {
                Map whole[NP];
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    whole[k] = maps[buf][0][k][lane];
#pragma unroll
                    for (int w = 1; w < kWarps; ++w) whole[k] = after(maps[buf][w][k][lane], whole[k]);
                }
                exchange<NP>(peers, bars, C, rank, s, whole, h, carry, to, lost);
            }
            if (p.chk != nullptr && tile < tiles) store_state<NP>(p.chk + (ch.slot0 + tile) * p.D + d, n, h);
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    start[buf][w][k][lane] = h[k];
                    h[k] = apply(maps[buf][w][k][lane], h[k]);
                }
            if (C == 1) {
#pragma unroll
                for (int k = 0; k < NP; ++k) carry[k] = h[k];
            }
            __syncwarp();
            if (lane == 0) arrive(&bars.start[buf]);
        }
        if (rank == 0) store_state<NP>(p.hlast + seq * p.D + d, n, carry);
    } else {
        // ---------------------------------------------------------------- the warps with a segment each
        const Constants k = constants();
        Pair nsp2[NP];
        decay_rates<NP>(p.lam + d, p.c * 1.4426950408889634f, n, nsp2);
        const bool slow = slow_decays<NP>(nsp2);
        const int row_bytes = min(Lanes<NP>::chans, p.D - ct * Lanes<NP>::chans) * (int)sizeof(T);
        const unsigned char* src[3];
        long long step[3];
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            src[q] = static_cast<const unsigned char*>(p.in[q].p) + (ch.b * p.in[q].sb + ch.t0 * p.in[q].st + ct * Lanes<NP>::chans) * (long long)sizeof(T);
            step[q] = p.in[q].st * (long long)sizeof(T);
        }
        const unsigned char* ring = smem + wid * R::ring;
        const uint32_t ring_at = smem_u32(ring);
        auto request = [&](int s, int stage) {
            const int row0 = (s * C + rank) * kTile + wid * TS;
            if (s < steps && row0 < ch.len) fetch<T, MIS, NP, false, 3>(ring_at + stage * R::stage, src, step, row0, ch.len - row0, row_bytes);
            cp_commit();
        };
#pragma unroll
        for (int s = 0; s < ST; ++s) request(s, s);

        int stage = 0;
        // the gates of tile s: coefficients of the segment and its map
        auto gates = [&](int s, Pair(&a)[TS][NP], Pair(&b)[TS][NP]) {
            const int row0 = (s * C + rank) * kTile + wid * TS, left = ch.len - row0;  // steps of the segment that exist: may be <= 0
            cp_wait<ST - 1>();
            __syncwarp();
            const unsigned char* st = ring + stage * R::stage;
            Map m[NP];
#pragma unroll
            for (int e = 0; e < NP; ++e) m[e] = {k.one, 0};
            auto work = [&](auto slow, bool whole) {  // both constants at every call
#pragma unroll
                for (int j = 0; j < TS; ++j) {
                    Pair x[NP], r[NP], i[NP];
                    auto read = [&](int q, Pair(&v)[NP]) {
                        row_lane<T, MIS, NP>(st + q * R::bytes + j * R::pitch, lane,
                                         MIS ? (uint32_t)(reinterpret_cast<uintptr_t>(src[q]) + (row0 + j) * step[q]) : 0u, v);
                    };
                    read(0, x), read(1, r), read(2, i);
#pragma unroll
                    for (int e = 0; e < NP; ++e) {
                        const Decay dec = decay2<decltype(slow)::value>(k, mul2(nsp2[e], sigmoid2(k, r[e])));
                        const float2 q = pair2(minus_beta2(dec.u));
                        a[j][e] = dec.a;
                        b[j][e] = mul2(mul2(bits2(make_float2(root(-q.x), root(-q.y))), x[e]), sigmoid2(k, i[e]));
                        if (!whole && j >= left) a[j][e] = k.one, b[j][e] = 0;
                        m[e].sum = fma2(a[j][e], m[e].sum, b[j][e]);
                        m[e].decay = mul2(m[e].decay, a[j][e]);
                    }
                }
            };
            if (slow && left >= TS) work(Bool<true>(), true);
            else work(Bool<false>(), false);
#pragma unroll
            for (int e = 0; e < NP; ++e) maps[s & 1][wid][e][lane] = m[e];
            __syncwarp();
            if (lane == 0) arrive(&bars.maps[s & 1]);
            request(s + ST, stage);
            stage = stage == ST - 1 ? 0 : stage + 1;
        };
        // the states of tile s, from the ones that enter the segment
        auto states = [&](int s, const Pair(&a)[TS][NP], const Pair(&b)[TS][NP]) {
            const int row0 = (s * C + rank) * kTile + wid * TS, left = ch.len - row0;
            T* out = static_cast<T*>(p.out[0]) + (ch.row0 + row0) * p.D + d;
            await(&bars.start[s & 1], (uint32_t)(s >> 1) & 1u, lost);
            Pair h[NP];
#pragma unroll
            for (int e = 0; e < NP; ++e) h[e] = start[s & 1][wid][e][lane];
#pragma unroll
            for (int j = 0; j < TS; ++j) {
#pragma unroll
                for (int e = 0; e < NP; ++e) h[e] = fma2(a[j][e], h[e], b[j][e]);
                if (j < left) store_lane<T, NP>(out, h, !MIS || p.whole, n);
                out += p.D;
            }
        };
        // The gates of the next tile are computed before the states of this one, with two tiles' coefficients in registers:
        // 8 x 4096 x 2048 float32 takes 207 us, 266 without. (The adjoint has twice as many coefficients and would spill: 560 us
        // against 360.)
        Pair a0[TS][NP], b0[TS][NP], a1[TS][NP], b1[TS][NP];
        for (int s = -1; s < steps; s += 2) {  // (each piece of code twice, not three times: the loop has to stay in the instruction cache)
            if (s + 1 < steps) gates(s + 1, a0, b0);
            if (s >= 0) states(s, a1, b1);
            if (s + 2 < steps) gates(s + 2, a1, b1);
            if (s + 1 < steps) states(s + 1, a0, b0);
        }
        cp_wait<0>();
    }
    __syncwarp();
    close_exchange(C, lost);
}

// ------------------------------------------------------------------------------------------- adjoint
// Tiles from the last to the first; CTA `rank` of a cluster takes the tile `rank` places before the newest. Inside a
// tile the states run forward from the kept state and the adjoint runs backward from the carry; both folds use the
// same products of decays, so a segment hands over one decay and two sums. Between CTAs only the adjoint's maps travel: every tile
// has its own kept state.
template <typename T, bool MIS, int NP>
__global__ void __launch_bounds__(kThreads, 2) gated_bwd_kernel(const Args p) {
    using R = Rows<T, MIS, NP, true>;
    constexpr int ST = Shape<true>::stages, TS = kSteps;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ Map maps[2][kWarps][NP][32];     // decays, sums of the adjoint
    __shared__ Pair sums[2][kWarps][NP][32];    // sums of the states
    __shared__ Map start[2][kWarps][NP][32];    // the state before a segment and the adjoint behind it
    Map(*const peers)[NP][32] = reinterpret_cast<Map(*)[NP][32]>(smem + kWarps * R::ring);  // [2 * C], in clusters only
    __shared__ __align__(8) Barriers bars;
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int C = p.C, rank = (int)(blockIdx.x % C);
    const long long chain = blockIdx.x / C;
    const int ct = (int)(chain % p.ctiles);
    const long long seq = chain / p.ctiles;
    if (seq == p.S) {
        clear_spare_rows<T, NP>(p, 3, ct, rank);
        return;
    }
    const Chain ch = locate(p, seq);
    const int d = ct * Lanes<NP>::chans + 2 * NP * lane, n = p.D - d;
    const int tiles = (ch.len + kTile - 1) / kTile, steps = (tiles + C - 1) / C;
    bool lost = false;
    Pair wsum[NP] = {};
    open_exchange(C, bars);

    if (wid == kWarps) {
        int to = C;
        Pair carry[NP] = {}, next[NP];
        if (p.glast != nullptr) load_state<NP>(p.glast + seq * p.D + d, n, carry);
        auto kept = [&](int s) {
            const int tile = tiles - 1 - (s * C + rank);
            if (s < steps && tile >= 0) load_state<NP>(p.chk + (ch.slot0 + tile) * p.D + d, n, next);
        };
#pragma unroll
        for (int k = 0; k < NP; ++k) next[k] = 0;
        kept(0);
        for (int s = 0; s < steps; ++s) {
            const int buf = s & 1;
            Pair h[NP], g[NP];
#pragma unroll
            for (int k = 0; k < NP; ++k) h[k] = next[k];
            kept(s + 1);
            await(&bars.maps[buf], (uint32_t)(s >> 1) & 1u, lost);
            if (C == 1) {
#pragma unroll
                for (int k = 0; k < NP; ++k) g[k] = carry[k];
            } else {
                Map whole[NP];
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    whole[k] = maps[buf][kWarps - 1][k][lane];
#pragma unroll
                    for (int w = kWarps - 2; w >= 0; --w) whole[k] = after(maps[buf][w][k][lane], whole[k]);
                }
                exchange<NP>(peers, bars, C, rank, s, whole, g, carry, to, lost);
            }
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                Pair before[kWarps];
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    before[w] = h[k];
                    h[k] = fma2(maps[buf][w][k][lane].decay, h[k], sums[buf][w][k][lane]);
                }
#pragma unroll
                for (int w = kWarps - 1; w >= 0; --w) {
                    start[buf][w][k][lane] = {before[w], g[k]};
                    g[k] = apply(maps[buf][w][k][lane], g[k]);
                }
                if (C == 1) carry[k] = g[k];
            }
            __syncwarp();
            if (lane == 0) arrive(&bars.start[buf]);
        }
        if (rank == 0 && p.hlast != nullptr) store_state<NP>(p.hlast + seq * p.D + d, n, carry);
    } else {
        const Constants k = constants();
        Pair nsp2[NP], nsp[NP], per_sp[NP];
        decay_rates<NP>(p.lam + d, p.c * 1.4426950408889634f, n, nsp2);
        decay_rates<NP>(p.lam + d, p.c, n, nsp);
        const bool slow = slow_decays<NP>(nsp2);
#pragma unroll
        for (int e = 0; e < NP; ++e) {
            const float2 sp = pair2(nsp[e]);
            per_sp[e] = bits2(make_float2(1.f / fminf(sp.x, -1.17549435e-38f), 1.f / fminf(sp.y, -1.17549435e-38f)));  // rho = l per_sp
        }
        const int row_bytes = min(Lanes<NP>::chans, p.D - ct * Lanes<NP>::chans) * (int)sizeof(T);
        const unsigned char* src[4];
        long long step[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            src[q] = static_cast<const unsigned char*>(p.in[q].p) + (ch.b * p.in[q].sb + ch.t0 * p.in[q].st + ct * Lanes<NP>::chans) * (long long)sizeof(T);
            step[q] = p.in[q].st * (long long)sizeof(T);
        }
        const unsigned char* ring = smem + wid * R::ring;
        const uint32_t ring_at = smem_u32(ring);
        auto first_row = [&](int s) { return (tiles - 1 - (s * C + rank)) * kTile + wid * TS; };
        auto request = [&](int s, int stage) {
            const int row0 = first_row(s);
            if (s < steps && row0 >= 0 && row0 < ch.len) fetch<T, MIS, NP, true, 4>(ring_at + stage * R::stage, src, step, row0, ch.len - row0, row_bytes);
            cp_commit();
        };
#pragma unroll
        for (int s = 0; s < ST; ++s) request(s, s);
        auto read = [&](int stage, int q, int row0, int j, Pair(&v)[NP]) {
            row_lane<T, MIS, NP>(ring + stage * R::stage + q * R::bytes + j * R::pitch, lane,
                             MIS ? (uint32_t)(reinterpret_cast<uintptr_t>(src[q]) + (row0 + j) * step[q]) : 0u, v);
        };
        struct Coeffs {
            Pair a[TS][NP], l[TS][NP], b[TS][NP], m[TS][NP];  // b = beta iota, m = -(a l / beta) iota
        };
        const Pair minus2 = resident(-2.f), tiny = resident(1.17549435e-38f);
        int stage = 0;
        auto gates = [&](int s, Coeffs& f) {
            const int row0 = first_row(s), left = row0 < 0 ? 0 : ch.len - row0;
            cp_wait<ST - 1>();
            __syncwarp();
            Pair A[NP], H[NP], G[NP];
#pragma unroll
            for (int e = 0; e < NP; ++e) A[e] = k.one, H[e] = 0, G[e] = 0;
            auto work = [&](auto slow, bool whole) {  // both constants at every call
#pragma unroll
                for (int j = 0; j < TS; ++j) {
                    Pair x[NP], r[NP], i[NP];
                    read(stage, 0, row0, j, x), read(stage, 1, row0, j, r), read(stage, 2, row0, j, i);
#pragma unroll
                    for (int e = 0; e < NP; ++e) {
                        const Pair rho = sigmoid2(k, r[e]), l = mul2(nsp[e], rho);
                        const auto [u, a] = decay2<decltype(slow)::value>(k, mul2(nsp2[e], rho));
                        // beta^2 and the smallest normal number, so that l / beta is 0 where l is
                        const Pair q = fma2(u, fma2(u, k.neg1, minus2), tiny);
                        const float2 b2 = pair2(q);
                        const Pair s = bits2(make_float2(rsq(b2.x), rsq(b2.y)));
                        const Pair si = mul2(s, sigmoid2(k, i[e]));
                        f.l[j][e] = l;
                        f.a[j][e] = a;
                        f.b[j][e] = mul2(q, si);
                        f.m[j][e] = mul2(mul2(a, mul2(l, k.neg1)), si);
                        Pair b = mul2(f.b[j][e], x[e]);
                        if (!whole && j >= left) f.a[j][e] = k.one, b = 0;
                        H[e] = fma2(f.a[j][e], H[e], b);
                        A[e] = mul2(A[e], f.a[j][e]);
                    }
                }
#pragma unroll
                for (int j = TS - 1; j >= 0; --j)
                    if (whole || j < left) {
                        Pair g[NP];
                        read(stage, 3, row0, j, g);
#pragma unroll
                        for (int e = 0; e < NP; ++e) G[e] = mul2(f.a[j][e], add2(g[e], G[e]));
                    }
            };
            if (slow && left >= TS) work(Bool<true>(), true);
            else work(Bool<false>(), false);
#pragma unroll
            for (int e = 0; e < NP; ++e) maps[s & 1][wid][e][lane] = {A[e], G[e]}, sums[s & 1][wid][e][lane] = H[e];
            __syncwarp();
            if (lane == 0) arrive(&bars.maps[s & 1]);
        };
        auto gradients = [&](int s, const Coeffs& f) {
            const int row0 = first_row(s), left = row0 < 0 ? 0 : ch.len - row0;
            await(&bars.start[s & 1], (uint32_t)(s >> 1) & 1u, lost);
            Pair g[NP], before[TS][NP], x[NP];
#pragma unroll
            for (int e = 0; e < NP; ++e) {
                const Map enter = start[s & 1][wid][e][lane];
                before[0][e] = enter.decay, g[e] = enter.sum;
            }
#pragma unroll
            for (int j = 0; j + 1 < TS; ++j) {
                read(stage, 0, row0, j, x);
#pragma unroll
                for (int e = 0; e < NP; ++e) before[j + 1][e] = fma2(f.a[j][e], before[j][e], mul2(f.b[j][e], x[e]));
            }
            long long o = (ch.row0 + row0 + TS - 1) * p.D + d;
#pragma unroll
            for (int j = TS - 1; j >= 0; --j) {
                if (j < left) {
                    Pair r[NP], i[NP], gh[NP], gx[NP], gr[NP], gi[NP];
                    read(stage, 0, row0, j, x), read(stage, 1, row0, j, r), read(stage, 2, row0, j, i), read(stage, 3, row0, j, gh);
#pragma unroll
                    for (int e = 0; e < NP; ++e) {
                        const Pair t = add2(gh[e], g[e]);
                        g[e] = mul2(f.a[j][e], t);
                        gx[e] = mul2(t, f.b[j][e]);
                        gi[e] = mul2(mul2(gx[e], x[e]), co_sigmoid2(k, i[e]));
                        const Pair w = mul2(g[e], fma2(f.m[j][e], x[e], mul2(f.l[j][e], before[j][e])));
                        wsum[e] = add2(wsum[e], w);
                        gr[e] = mul2(w, complement2(k, r[e], mul2(f.l[j][e], per_sp[e])));
                    }
                    store_lane<T, NP>(static_cast<T*>(p.out[0]) + o, gx, !MIS || p.whole, n);
                    store_lane<T, NP>(static_cast<T*>(p.out[1]) + o, gr, !MIS || p.whole, n);
                    store_lane<T, NP>(static_cast<T*>(p.out[2]) + o, gi, !MIS || p.whole, n);
                }
                o -= p.D;
            }
            __syncwarp();  // the rows have been read by all lanes
            request(s + ST, stage);
            stage = stage == ST - 1 ? 0 : stage + 1;
        };
        Coeffs f;
        for (int s = 0; s < steps; ++s) {
            gates(s, f);
            gradients(s, f);
        }
        cp_wait<0>();
    }
    __syncwarp();
    close_exchange(C, lost);
    if (wid < kWarps)
#pragma unroll
        for (int e = 0; e < NP; ++e) sums[0][wid][e][lane] = wsum[e];
    __syncthreads();
    if (wid == 0) {
#pragma unroll
        for (int e = 0; e < NP; ++e)
            for (int w = 1; w < kWarps; ++w) wsum[e] = add2(wsum[e], sums[0][w][e][lane]);
        store_state<NP>(p.part + (seq * C + rank) * p.D + d, n, wsum);
    }
}

// Sums of part[rows, D] over its rows in a fixed order: 32 channels per block, 32 threads per channel each adding every
// 32nd row of the block's share; `last`: the sums are the gradients of lam, scaled by sigmoid(lam) / softplus(lam).
__global__ void __launch_bounds__(1024) gated_lam_kernel(const float* __restrict__ part, long long rows, int D, float* __restrict__ out,
                                                         const float* __restrict__ lam, int last) {
    __shared__ float red[32][33];
    const int dl = threadIdx.x & 31, k = threadIdx.x >> 5, d = blockIdx.x * 32 + dl;
    const long long share = (rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * share, r1 = min(rows, r0 + share);
    float s = 0.f;
    if (d < D)
        for (long long r = r0 + k; r < r1; r += 32) s += part[r * D + d];
    red[k][dl] = s;
    __syncthreads();
    if (k == 0 && d < D) {
        s = 0.f;
        for (int j = 0; j < 32; ++j) s += red[j][dl];
        if (last) {
            // sigmoid(lam) / softplus(lam) is 1 - e^lam / 2 and less: one to the last bit below -17, where either underflows later on
            const float v = lam[d];
            out[d] = s * (v < -17.f ? 1.f : 1.f / (1.f + expf(-v)) / softplus(v));
        } else {
            out[(long long)blockIdx.y * D + d] = s;
        }
    }
}

// ------------------------------------------------------------------------------------------- one token per row
// Row b takes the state of its slot and writes it back. A slot that is named twice is worked off in row order by its
// first row; a slot outside the cache (-1: an empty row of a padded batch) leaves the cache alone and yields zeros. Four
// channels per thread; every warp looks through the slots by itself, which needs no barrier. Bound by latency for a few
// rows (the launch: 5.3 us a call), by HBM for many: 256 x 4096 bfloat16 8.2 us with four channels per thread, 10.2 with one.
struct StepArgs {
    Seq in[3];
    void* out;
    const float* lam;
    float* state;
    long long state_pitch;
    const void* slots;
    int slots64;
    long long B, n;
    int D;
    float c;
    int whole;  // four channels of every operand can be read and written at a time
};
constexpr int kStepThreads = 128, kStepChans = 4;

// softplus for one use: log(1 + e) as 2 atanh(e / (2 + e)), the series to the 13th power (the argument is at most 1/3: 2e-8)
__device__ __forceinline__ float softplus_once(float x) {
    const float e = ex2(-1.4426950408889634f * fabsf(x)), s = e * rcp(2.f + e), q = s * s;
    float t = fmaf(q, 1.f / 13.f, 1.f / 11.f);
    t = fmaf(q, t, 1.f / 9.f);
    t = fmaf(q, t, 1.f / 7.f);
    t = fmaf(q, t, 1.f / 5.f);
    t = fmaf(q, t, 1.f / 3.f);
    return fmaxf(x, 0.f) + 2.f * fmaf(s * q, t, s);
}

template <typename T>
__global__ void __launch_bounds__(kStepThreads) gated_step_kernel(const StepArgs p) {
    constexpr int V = kStepChans;
    const long long b = blockIdx.y;
    const int d = (blockIdx.x * kStepThreads + threadIdx.x) * V, n = p.D - d;  // this thread's first channel, and how many from it on
    auto slot_of = [&](long long row) -> long long {
        if (p.slots == nullptr) return row;
        return p.slots64 ? static_cast<const long long*>(p.slots)[row] : (long long)static_cast<const int*>(p.slots)[row];
    };
    auto load = [&](int q, long long row, Pair(&v)[2]) {
        const T* e = static_cast<const T*>(p.in[q].p) + row * p.in[q].sb + d;
        if (p.whole) {
            if (n <= 0) {
                v[0] = v[1] = 0;
            } else if constexpr (sizeof(T) == 4) {
                const float4 f = *reinterpret_cast<const float4*>(e);
                v[0] = bits2(make_float2(f.x, f.y)), v[1] = bits2(make_float2(f.z, f.w));
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(e);
                v[0] = bits2(unpack(w.x, T())), v[1] = bits2(unpack(w.y, T()));
            }
        } else {
            float f[V];
#pragma unroll
            for (int k = 0; k < V; ++k) f[k] = k < n ? to_float(e[k]) : 0.f;
            v[0] = bits2(make_float2(f[0], f[1])), v[1] = bits2(make_float2(f[2], f[3]));
        }
    };
    const long long slot = slot_of(b);
    const bool have = slot >= 0 && slot < p.n;
    Pair x[2], r[2], i[2], h[2] = {}, nsp2[2];
    load(0, b, x), load(1, b, r), load(2, b, i);
    float* at = p.state + (have ? slot : 0) * p.state_pitch + d;
    if (have) {
        if (p.whole && n > 0) {
            const float4 f = *reinterpret_cast<const float4*>(at);
            h[0] = bits2(make_float2(f.x, f.y)), h[1] = bits2(make_float2(f.z, f.w));
        } else {
            load_state<2>(at, n, h);
        }
    }
    load_state<2>(p.lam + d, n, nsp2);
    bool later = false;
    if (p.slots != nullptr && p.B > 1 && have) {  // `have` and `slot` are the block's
        bool earlier = false;
        for (long long j = threadIdx.x & 31; j < p.B; j += 32)
            if (slot_of(j) == slot) earlier |= j < b, later |= j > b;
        if (__any_sync(0xffffffffu, earlier)) return;  // the slot's first row does this one too
        later = __any_sync(0xffffffffu, later);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const float2 l = pair2(nsp2[e]);
        nsp2[e] = mul2(bits2(make_float2(softplus_once(l.x), softplus_once(l.y))), bits2(both(-1.4426950408889634f * p.c)));
    }
    const Constants k = constants();
    for (long long row = b;;) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const auto [u, a] = decay2<false>(k, mul2(nsp2[e], sigmoid2(k, r[e])));
            const float2 q = pair2(minus_beta2(u));
            const Pair beta = bits2(make_float2(root(-q.x), root(-q.y)));
            h[e] = fma2(a, h[e], mul2(mul2(beta, sigmoid2(k, i[e])), x[e]));
        }
        const Pair y[2] = {have ? h[0] : 0, have ? h[1] : 0};
        T* out = static_cast<T*>(p.out) + row * p.D + d;
        if constexpr (sizeof(T) == 4) {
            if (p.whole) {
                const float2 lo = pair2(y[0]), hi = pair2(y[1]);
                if (n > 0) *reinterpret_cast<float4*>(out) = make_float4(lo.x, lo.y, hi.x, hi.y);
            } else {
                store_state<2>(out, n, y);
            }
        } else {
            store_lane<T, 2>(out, y, p.whole != 0, n);
        }
        if (!later) break;
        do ++row;
        while (row < p.B && slot_of(row) != slot);
        if (row >= p.B) break;
        load(0, row, x), load(1, row, r), load(2, row, i);
    }
    if (have) {
        if (p.whole) {
            const float2 lo = pair2(h[0]), hi = pair2(h[1]);
            if (n > 0) *reinterpret_cast<float4*>(at) = make_float4(lo.x, lo.y, hi.x, hi.y);
        } else {
            store_state<2>(at, n, h);
        }
    }
}

// ------------------------------------------------------------------------------------------- host
// How a call is cut up: pairs of channels per lane, chains of a sequence, CTAs per chain. Two CTAs fit on an SM (but for the
// adjoint of 16 bits with two pairs per lane and clusters of twelve, 118 KB each: one), and one round of them is best: the
// largest of 1, 2, 4, 8 and 12 CTAs per chain that stays within 2 x 148 (8 x 4096 x 2048 bf16, 128 chains, forward and adjoint: 595 us
// with one, 473 with two, 530 with three, 489 with four; 65536 x 1024, 16 chains: 1010 with eight, 722 with twelve, 947 with sixteen,
// which few GPCs can hold twice). Packed sequences differ in length, and several rounds even them out (23 of 0 to 3000 steps, 368
// chains: 349 us with one CTA, 239 with four). Chains in 16 bits are 128 channels wide (10 x 1500 x 700: 144 us against 170 with 64),
// or 64 where those would be too few.
struct Cut {
    int np, ctiles, C;
};
inline Cut cut(int dtype, long long S, long long rows, int D, bool packed) {
    Cut c = {dtype == B200_F32 ? 1 : 2, 0, 1};
    const long long tiles = S > 0 ? (rows / S + kTile - 1) / kTile : 0, most = tiles < kMaxCluster ? tiles : kMaxCluster;
    if (c.np == 2 && S * ((D + 127) / 128) * most < 200) c.np = 1;
    c.ctiles = (D + 64 * c.np - 1) / (64 * c.np);
    const long long chains = S * c.ctiles, limit = (packed && S > 1 ? 5 : 1) * 2 * 148;
    for (int C : {2, 4, 8, 12})
        if (C <= most && chains * C <= limit) c.C = C;
    return c;
}
inline long long slots(long long S, long long L, long long T, bool packed) { return packed ? T / kTile + S + 1 : S * ((L + kTile - 1) / kTile); }

template <typename K>
int launch(K kernel, const Args& p, long long chains, size_t smem, cudaStream_t st) {
    const long long grid = chains * p.C;
    if (grid > 0x7fffffffLL) return B200_ERR_UNSUPPORTED;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return B200_ERR_LAUNCH;
    if (p.C > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return B200_ERR_LAUNCH;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned int)grid), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned int)p.C, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? B200_OK : B200_ERR_LAUNCH;
}

template <typename T, bool MIS, int NP>
int launch_as(bool bwd, const Args& p, long long chains, cudaStream_t st) {
    const size_t smem = (size_t)kWarps * (bwd ? Rows<T, MIS, NP, true>::ring : Rows<T, MIS, NP, false>::ring) +
                        (p.C > 1 ? 2 * p.C * NP * 32 * sizeof(Map) : 0);
    return bwd ? launch(gated_bwd_kernel<T, MIS, NP>, p, chains, smem, st) : launch(gated_fwd_kernel<T, MIS, NP>, p, chains, smem, st);
}
template <typename T>
int launch_typed(bool bwd, bool mis, int np, const Args& p, long long chains, cudaStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (np == 2) return mis ? launch_as<T, true, 2>(bwd, p, chains, st) : launch_as<T, false, 2>(bwd, p, chains, st);
    return mis ? launch_as<T, true, 1>(bwd, p, chains, st) : launch_as<T, false, 1>(bwd, p, chains, st);
}

inline int dispatch(int dtype, bool bwd, Args& p, long long S, long long rows, cudaStream_t st) {
    const int e = block_elem_size(dtype), n = bwd ? 4 : 3;
    const Cut c = cut(dtype, S, rows, p.D, p.cu != nullptr);
    p.ctiles = c.ctiles, p.C = c.C;
    bool mis = false;
    for (int q = 0; q < n; ++q) {
        if ((uintptr_t)p.in[q].p % e) return B200_ERR_ARG;
        mis |= (uintptr_t)p.in[q].p % 16 || (p.in[q].sb * e) % 16 || (p.in[q].st * e) % 16;
    }
    const int lane = 2 * c.np * e;  // bytes of a lane's channels
    p.whole = p.D * e % lane == 0;
    for (int q = 0; q < (bwd ? 3 : 1); ++q) {
        if ((uintptr_t)p.out[q] % e) return B200_ERR_ARG;
        p.whole = p.whole && (uintptr_t)p.out[q] % lane == 0;
    }
    mis |= !p.whole;  // the aligned kernels store a lane's channels at a time
    const long long chains = (S + (p.cu != nullptr ? 1 : 0)) * p.ctiles;
    if (dtype == B200_F32) return launch_typed<float>(bwd, mis, c.np, p, chains, st);
    if (dtype == B200_BF16) return launch_typed<__nv_bfloat16>(bwd, mis, c.np, p, chains, st);
    return launch_typed<__half>(bwd, mis, c.np, p, chains, st);
}

inline bool sizes_ok(int dtype, int64_t S, int64_t L, int64_t T, int64_t D) {
    return block_elem_size(dtype) != 0 && S >= 0 && L >= 0 && T >= 0 && L < (1LL << 30) && T < (1LL << 30) && D >= 1 && D <= (1 << 24);
}

struct Workspace {
    size_t part2, total;
    long long rows;
    int split;
};
inline Workspace plan(int dtype, long long S, long long L, long long T, int D, bool packed) {
    Workspace w;
    w.rows = S * cut(dtype, S, packed ? T : S * L, D, packed).C;
    // one block adds up to 1024 rows of 32 channels; more rows are added in two rounds
    w.split = (int)(w.rows <= 1024 ? 1 : w.rows / 512 < 256 ? w.rows / 512 : 256);
    w.part2 = align_up((size_t)w.rows * D * 4, 256);
    w.total = w.part2 + align_up(w.split > 1 ? (size_t)w.split * D * 4 : 0, 256) + 256;
    return w;
}

}  // namespace gated
namespace quant {
int product_status(cudaStream_t st);
}
}  // namespace b200

extern "C" {

int b200_block_status(void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int gated = b200::take_error_word(b200::gated::exchange_lost, st), product = b200::quant::product_status(st);
    return gated != B200_OK ? gated : product;
}

int64_t b200_gated_chk_rows(int dtype, int64_t S, int64_t L, int64_t T, int packed) {
    if (b200::block_elem_size(dtype) == 0 || S < 0 || L < 0 || T < 0) return 0;
    return b200::gated::slots(S, L, T, packed != 0);
}

int b200_gated_fwd(int dtype, int64_t S, int64_t L, int64_t T, int64_t D, float c, const void* cu, int cu_is64, const void* x, int64_t xb,
                   int64_t xt, const void* r, int64_t rb, int64_t rt, const void* i, int64_t ib, int64_t it, const void* lam, const void* h0,
                   void* h, void* hlast, void* chk, void* stream) {
    return b200_gated_probe(-1, dtype, S, L, T, D, c, cu, cu_is64, x, xb, xt, r, rb, rt, i, ib, it, lam, h0, h, hlast, chk, stream);
}

int b200_gated_probe(int mute_step, int dtype, int64_t S, int64_t L, int64_t T, int64_t D, float c, const void* cu, int cu_is64, const void* x,
                     int64_t xb, int64_t xt, const void* r, int64_t rb, int64_t rt, const void* i, int64_t ib, int64_t it, const void* lam,
                     const void* h0, void* h, void* hlast, void* chk, void* stream) {
    using namespace b200;
    using namespace b200::gated;
    if (!sizes_ok(dtype, S, L, T, D)) return B200_ERR_ARG;
    const bool packed = cu != nullptr;
    const long long rows = packed ? T : S * L;
    if (S == 0 && rows == 0) return B200_OK;
    if (!lam || (S > 0 && !hlast) || (rows > 0 && (!x || !r || !i || !h))) return B200_ERR_ARG;
    if (!on_boundary(4, lam, h0, hlast, chk) || !on_boundary(cu_is64 ? 8 : 4, cu)) return B200_ERR_ARG;
    Args p = {};
    p.in[0] = {x, xb, xt}, p.in[1] = {r, rb, rt}, p.in[2] = {i, ib, it};
    p.out[0] = h, p.lam = (const float*)lam, p.h0 = (const float*)h0, p.hlast = (float*)hlast, p.chk = (float*)chk;
    p.cu = cu, p.cu64 = cu_is64, p.S = S, p.L = L, p.T = T, p.D = (int)D, p.c = c;
    p.until = mute_step < 0 ? 0x7fffffff : mute_step;
    return dispatch(dtype, false, p, S, rows, static_cast<cudaStream_t>(stream));
}

size_t b200_gated_bwd_workspace_bytes(int dtype, int64_t S, int64_t L, int64_t T, int64_t D, int packed) {
    if (!b200::gated::sizes_ok(dtype, S, L, T, D)) return 256;
    return b200::gated::plan(dtype, S, L, T, (int)D, packed != 0).total;
}

int b200_gated_bwd(int dtype, int64_t S, int64_t L, int64_t T, int64_t D, float c, const void* cu, int cu_is64, const void* x, int64_t xb,
                   int64_t xt, const void* r, int64_t rb, int64_t rt, const void* i, int64_t ib, int64_t it, const void* lam, const void* chk,
                   const void* gh, int64_t gb, int64_t gt, const void* glast, void* gx, void* gr, void* gi, void* glam, void* gh0,
                   void* workspace, size_t workspace_bytes, void* stream) {
    using namespace b200;
    using namespace b200::gated;
    if (!sizes_ok(dtype, S, L, T, D)) return B200_ERR_ARG;
    const bool packed = cu != nullptr;
    const long long rows = packed ? T : S * L;
    if (!lam || !glam || (rows > 0 && (!x || !r || !i || !gh || !gx || !gr || !gi || !chk))) return B200_ERR_ARG;
    if (!on_boundary(4, lam, chk, glast, glam, gh0) || !on_boundary(cu_is64 ? 8 : 4, cu)) return B200_ERR_ARG;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (S == 0 && rows == 0) return cudaMemsetAsync(glam, 0, (size_t)D * 4, st) == cudaSuccess ? B200_OK : B200_ERR_LAUNCH;
    const Workspace w = plan(dtype, S, L, T, (int)D, packed);
    if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < w.total) return B200_ERR_WORKSPACE;
    Args p = {};
    p.in[0] = {x, xb, xt}, p.in[1] = {r, rb, rt}, p.in[2] = {i, ib, it}, p.in[3] = {gh, gb, gt};
    p.out[0] = gx, p.out[1] = gr, p.out[2] = gi;
    p.lam = (const float*)lam, p.hlast = (float*)gh0, p.glast = (const float*)glast, p.chk = (float*)const_cast<void*>(chk);
    p.part = (float*)workspace;
    p.cu = cu, p.cu64 = cu_is64, p.S = S, p.L = L, p.T = T, p.D = (int)D, p.c = c;
    const int rc = dispatch(dtype, true, p, S, rows, st);
    if (rc != B200_OK) return rc;
    float* part2 = (float*)((char*)workspace + w.part2);
    const unsigned int blocks = (unsigned int)((D + 31) / 32);
    if (w.split > 1) gated_lam_kernel<<<dim3(blocks, w.split), 1024, 0, st>>>(p.part, w.rows, (int)D, part2, p.lam, 0);
    gated_lam_kernel<<<dim3(blocks, 1), 1024, 0, st>>>(w.split > 1 ? part2 : p.part, w.split > 1 ? w.split : w.rows, (int)D, (float*)glam, p.lam, 1);
    return cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_LAUNCH;
}

int b200_gated_step(int dtype, int64_t B, int64_t D, int64_t n, float c, const void* x, int64_t xb, const void* r, int64_t rb, const void* i,
                    int64_t ib, const void* lam, void* state, int64_t state_pitch, const void* slots, int slots_are64, void* h, void* stream) {
    using namespace b200;
    using namespace b200::gated;
    const int e = block_elem_size(dtype);
    if (e == 0 || B < 0 || n < 0 || D < 1 || D > (1 << 24) || state_pitch < D) return B200_ERR_ARG;
    if (B == 0) return B200_OK;
    if (!x || !r || !i || !lam || !h || (n > 0 && !state) || (!slots && n < B)) return B200_ERR_ARG;
    if (!on_boundary(e, h) || !on_boundary(4, lam, state) || !on_boundary(slots_are64 ? 8 : 4, slots)) return B200_ERR_ARG;
    if (B > 65535) return B200_ERR_UNSUPPORTED;
    StepArgs p = {};
    p.in[0] = {x, xb, 0}, p.in[1] = {r, rb, 0}, p.in[2] = {i, ib, 0};
    p.out = h, p.lam = (const float*)lam, p.state = (float*)state, p.state_pitch = state_pitch;
    p.slots = slots, p.slots64 = slots_are64, p.B = B, p.n = n, p.D = (int)D, p.c = c;
    p.whole = D % kStepChans == 0 && (uintptr_t)h % (kStepChans * e) == 0 && (uintptr_t)state % 16 == 0 && state_pitch % 4 == 0;
    for (int q = 0; q < 3; ++q) {
        if ((uintptr_t)p.in[q].p % e) return B200_ERR_ARG;
        p.whole = p.whole && (uintptr_t)p.in[q].p % (kStepChans * e) == 0 && p.in[q].sb % kStepChans == 0;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned int)((D + kStepChans * kStepThreads - 1) / (kStepChans * kStepThreads)), (unsigned int)B);
    if (dtype == B200_F32) gated_step_kernel<float><<<grid, kStepThreads, 0, st>>>(p);
    else if (dtype == B200_BF16) gated_step_kernel<__nv_bfloat16><<<grid, kStepThreads, 0, st>>>(p);
    else gated_step_kernel<__half><<<grid, kStepThreads, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_LAUNCH;
}

}  // extern "C"
