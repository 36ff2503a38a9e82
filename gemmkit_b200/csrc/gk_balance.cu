// gk_balance.cu -- a router's balance loss, the experts' counts and offsets, and the loss's gradient.
//
//   p_te = softmax of token t's logits;  P_e = mean of p_te over the live tokens;  f_e = counts_e / routed
//   loss = coef E sum_e f_e P_e;   dloss/dlogit_te = rates_e-weighted:  p_te (rates_e - sum_j p_tj rates_j),
//   rates_e = coef E f_e / live
//
// Bound by memory: the logits are read once in each direction. A few lanes take a token, its logits in
// registers, and in the forward pass add its p to sums that stay in registers over all of their tokens;
// counts are integers in shared memory. Each block leaves its sums and counts, and a second kernel adds
// them (one block does all of it where there are few tokens). No floating atomics: which token a warp
// takes depends on the sizes (and the SMs) alone, and so does every sum.
// Differences of logits go through the fast exponential (2^-22, and 2^-24 of the difference: the large p
// come from small differences), sums over blocks through f64.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "gemmkit_cuda.h"
#include "gk_engine.h"
#include "gk_f2.cuh"
#include "gk_launch.h"
#include "gk_sm100.cuh"
#include "gk_store.cuh"

namespace gk {

namespace {

constexpr int MAX_EXPERTS = 1024;
constexpr int BW = 16;           // warps of a block

struct Router {
    const void* x;
    int64_t rs, cs;
    int32_t ids64;
    const void* ids;
    int32_t top, tokens, experts;
    unsigned int* status;
};

// How a warp takes tokens: L lanes a token, 32 / L tokens at a time, and lane q of a token's holds the logits
// (L j + q) V .. + V - 1 for j < J, as they lie: f32 bits, or 16-bit values two a word (V = 4) or one.
// (A whole warp a token spends most of its instructions on reductions over lanes: 155 a token of 256
// experts forward and 220 backward.)
template <int T_, int V_, int J_, int L_>
struct Layout {
    static constexpr int T = T_, V = V_, J = J_, L = L_, N = J * V, G = 32 / L;
    static constexpr int U = 1;  // tokens of a lane at a time, their loads in flight
};

template <typename C>
struct Logits {
    static constexpr int T = C::T, V = C::V, J = C::J;
    uint32_t w[C::N];
    __device__ __forceinline__ void load(const Router& p, int64_t t, int q) {
        constexpr int ES = T == GK_F32 ? 4 : 2;
        const uint8_t* row = static_cast<const uint8_t*>(p.x) + (t * p.rs + (V == 4 ? q * V : 0)) * ES;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int e = (C::L * j + q) * V;
            if (e >= p.experts) continue;
            if constexpr (V == 1) {
                const uint8_t* at = row + e * p.cs * ES;
                if (T == GK_F32)
                    w[j] = *reinterpret_cast<const uint32_t*>(at);
                else
                    w[j] = *reinterpret_cast<const uint16_t*>(at);
            } else if (T == GK_F32) {
                const uint4 v = ld_global_v4(row + C::L * j * V * ES);
                w[4 * j] = v.x, w[4 * j + 1] = v.y, w[4 * j + 2] = v.z, w[4 * j + 3] = v.w;
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(row + C::L * j * V * ES);
                w[4 * j] = v.x, w[4 * j + 1] = v.y;
            }
        }
    }
    __device__ __forceinline__ float value(int j, int v) const {
        if (T == GK_F32) return __uint_as_float(w[V * j + v]);
        const uint32_t h = V == 1 ? w[j] : w[V * j + v / 2] >> (16 * (v & 1));
        return T == GK_F16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xFFFFu)))
                           : __uint_as_float(h << 16);
    }
    // The softmax is y times the value returned; 0 everywhere where every logit is minus infinity.
    __device__ __forceinline__ float softmax(const Router& p, int q, F2 (&y)[C::N / 2]) const {
        float x[C::N], m = -INFINITY;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                x[V * j + v] = (C::L * j + q) * V < p.experts ? value(j, v) : -INFINITY;
                m = fmaxf(m, x[V * j + v]);
            }
#pragma unroll
        for (int d = C::L / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        const bool none = m == -INFINITY;
        // (the difference first: logits of the type's lowest value stay apart from infinities)
        const F2 scale(1.44269504f), base(none ? 0.0f : -m);
        F2 s2(0.0f);
#pragma unroll
        for (int i = 0; i < C::N / 2; ++i) {
            const F2 t = mul2(add2(F2(x[2 * i], x[2 * i + 1]), base), scale);
            y[i] = F2(exp2_hw(t.lo()), exp2_hw(t.hi()));
            s2 = add2(s2, y[i]);
        }
        float s = s2.lo() + s2.hi();
#pragma unroll
        for (int d = C::L / 2; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        // (a row of NaN also has no maximum: its sum is NaN, and stays so)
        return none && s == 0.0f ? 0.0f : __frcp_rn(s);
    }
};

// A token's ids into `hist` (when there is one), its L lanes together; whether it has any. All lanes of the
// warp call it, with on == false where they have no token.
template <int L>
__device__ __forceinline__ bool token_ids(const Router& p, int64_t t, bool on, int* hist, int lane) {
    const int q = lane % L;
    bool any = false, bad = false;
    for (int i = q; on && i < p.top; i += L) {
        const int64_t at = t * p.top + i;
        const int64_t id = p.ids64 ? static_cast<const int64_t*>(p.ids)[at]
                                   : static_cast<const int32_t*>(p.ids)[at];
        if (id >= 0 && id < p.experts) {
            any = true;
            if (hist) atomicAdd(&hist[id], 1);
        } else if (id >= 0) {
            bad = true;
        }
    }
    if (hist && bad) atomicOr(p.status, GK_DEV_BAD_OFFSETS);
    const uint32_t who = __ballot_sync(0xffffffffu, any);
    constexpr uint32_t mine = L == 32 ? 0xffffffffu : (1u << (L & 31)) - 1u;
    return (who >> (lane - q) & mine) != 0;
}

// What a block leaves, in words: experts sums (f32), experts counts and the live tokens. Behind all
// blocks' parts, in whole 16-byte pieces, lie their totals: experts sums (f64), experts counts, the live
// tokens and the blocks of the second kernel that are done.
__host__ __device__ inline int part_pitch(int experts) { return 2 * experts + 1; }
__host__ __device__ inline int64_t totals_at(int blocks, int experts) {
    return (static_cast<int64_t>(blocks) * part_pitch(experts) + 3) / 4 * 4;
}
__host__ __device__ inline int64_t part_words(int blocks, int experts) {
    return totals_at(blocks, experts) + 3 * experts + 2;
}

struct BalanceOut {
    float coef;
    float* loss;
    int32_t* counts;
    int32_t* offsets;
    float* rates;
};

// The results from the totals; sum(e) and count(e) give an expert's. All threads of a block of W warps.
template <int W, typename S, typename N>
__device__ __forceinline__ void finish(S sum, N count, int tokens, int experts, const BalanceOut& o) {
    __shared__ double red[W];
    __shared__ int scan[W];
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    constexpr int PER = MAX_EXPERTS / (32 * W);  // thread e, and e + 32 W
    int cnt[PER], routed = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int e = k * 32 * W + tid;
        const int c = e < experts ? count(e) : 0;
        cnt[k] = c;
        int inc = c;  // running sums of the counts
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += u;
        }
        if (lane == 31) scan[w] = inc;
        __syncthreads();
        int before = routed;
        for (int i = 0; i < w; ++i) before += scan[i];
        if (e < experts) {
            o.counts[e] = c;
            o.offsets[e + 1] = before + inc;
        }
        for (int i = 0; i < W; ++i) routed += scan[i];
        __syncthreads();
    }
    if (tid == 0) o.offsets[0] = 0;
    double a = 0.0;
    const double unit =
        routed > 0 ? static_cast<double>(o.coef) * experts / routed / tokens : 0.0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int e = k * 32 * W + tid;
        if (e < experts) {
            o.rates[e] = static_cast<float>(unit * cnt[k]);
            if (routed > 0) a += unit * cnt[k] * sum(e);
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) a += __shfl_xor_sync(0xffffffffu, a, d);
    if (lane == 0) red[w] = a;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < W; ++i) a += red[i];
        *o.loss = static_cast<float>(a);
    }
}

template <typename C>
__global__ void __launch_bounds__(32 * BW, C::N <= 16 ? 2 : 1)
    balance_kernel(const Router p, uint32_t* part, const BalanceOut o) {
    extern __shared__ float smem[];  // BW x experts sums, then the block's part
    uint32_t* own = reinterpret_cast<uint32_t*>(smem + BW * p.experts);
    int* hist = reinterpret_cast<int*>(own + p.experts);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, q = lane % C::L;
    for (int i = threadIdx.x; i <= p.experts; i += blockDim.x) hist[i] = 0;  // counts, live tokens
    griddep_wait();
    griddep_launch_dependents();
    __syncthreads();
    F2 sum[C::N / 2];
#pragma unroll
    for (int i = 0; i < C::N / 2; ++i) sum[i] = F2(0.0f);
    int live = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * BW * C::G * C::U;
    for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * BW + w) * C::G * C::U; t0 < p.tokens; t0 += step) {
        Logits<C> x[C::U];
#pragma unroll
        for (int k = 0; k < C::U; ++k) {
            const int64_t t = t0 + k * C::G + lane / C::L;
            if (t < p.tokens) x[k].load(p, t, q);
        }
#pragma unroll
        for (int k = 0; k < C::U; ++k) {
            const int64_t t = t0 + k * C::G + lane / C::L;
            const bool has = token_ids<C::L>(p, t, t < p.tokens, hist, lane);
            live += has && q == 0;
            if (!__any_sync(0xffffffffu, has)) continue;
            F2 y[C::N / 2];
            const float inv = x[k].softmax(p, q, y);
            if (has) {  // (padding may hold anything)
#pragma unroll
                for (int i = 0; i < C::N / 2; ++i) sum[i] = fma2(y[i], F2(inv), sum[i]);
            }
        }
    }
    live = __reduce_add_sync(0xffffffffu, live);
    // the warp's sums: the tokens that it took at one time lie L lanes apart
#pragma unroll
    for (int j = 0; j < C::J; ++j)
#pragma unroll
        for (int v = 0; v < C::V; ++v) {
            const F2 pair = sum[(C::V * j + v) / 2];
            float a = (C::V * j + v) & 1 ? pair.hi() : pair.lo();
#pragma unroll
            for (int d = C::L; d < 32; d <<= 1) a += __shfl_xor_sync(0xffffffffu, a, d);
            const int e = (C::L * j + q) * C::V + v;
            if (lane < C::L && e < p.experts) smem[w * p.experts + e] = a;
        }
    if (lane == 0 && live) atomicAdd(&hist[p.experts], live);
    __syncthreads();
    for (int e = threadIdx.x; e < p.experts; e += blockDim.x) {
        float a = smem[e];
#pragma unroll
        for (int i = 1; i < BW; ++i) a += smem[i * p.experts + e];
        own[e] = __float_as_uint(a);
    }
    __syncthreads();
    if (gridDim.x == 1) {
        finish<BW>([&](int e) { return static_cast<double>(__uint_as_float(own[e])); },
               [&](int e) { return hist[e]; }, hist[p.experts], p.experts, o);
        return;
    }
    const int pitch = part_pitch(p.experts);
    for (int i = threadIdx.x; i < pitch; i += blockDim.x)
        part[static_cast<int64_t>(blockIdx.x) * pitch + i] = own[i];
    if (blockIdx.x == 0 && threadIdx.x == 0)
        part[totals_at(gridDim.x, p.experts) + 3 * p.experts + 1] = 0;
}

// The parts of `blocks` blocks: a block adds 32 experts', a thread every FW-th part's, in f64; the block
// that is done last turns the totals into the results. (One block for all parts took 34 us for
// 148 x 256, a chain of 148 additions in f64.)
constexpr int FW = 32;

__global__ void __launch_bounds__(32 * FW)
    balance_finish_kernel(uint32_t* part, int blocks, int experts, const BalanceOut o) {
    __shared__ double s[FW][32];
    __shared__ int c[FW][32];
    __shared__ int last;
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int pitch = part_pitch(experts), e = blockIdx.x * 32 + lane;
    uint32_t* totals = part + totals_at(blocks, experts);
    double* sums = reinterpret_cast<double*>(totals);
    int* counts = reinterpret_cast<int*>(totals + 2 * experts);
    double a = 0.0;
    int n = 0, live = 0;
#pragma unroll 10
    for (int b = w; b < blocks; b += FW) {
        const uint32_t* at = part + static_cast<int64_t>(b) * pitch;
        if (e < experts) {
            a += static_cast<double>(__uint_as_float(at[e]));
            n += static_cast<int>(at[experts + e]);
        }
        if (blockIdx.x == 0) live += static_cast<int>(at[2 * experts]);
    }
    s[w][lane] = a;
    c[w][lane] = n;
    __syncthreads();
    if (w == 0 && e < experts) {
        for (int i = 1; i < FW; ++i) {
            a += s[i][lane];
            n += c[i][lane];
        }
        sums[e] = a;
        counts[e] = n;
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        if (lane == 0) c[w][0] = live;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int i = 1; i < FW; ++i) live += c[i][0];
            counts[experts] = live;
        }
    }
    if (w == 0) __threadfence();  // what this warp wrote, before the count
    __syncthreads();
    if (threadIdx.x == 0)
        last = atomicAdd(reinterpret_cast<unsigned*>(counts + experts + 1), 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    finish<FW>([&](int i) { return __ldcg(sums + i); }, [&](int i) { return __ldcg(counts + i); },
           __ldcg(counts + experts), experts, o);
}

template <typename C>
__global__ void __launch_bounds__(256, C::N <= 16 ? 4 : 2)
    balance_backward_kernel(const Router p, const float* rates, const float* dloss, void* dx,
                            int64_t ds, int64_t dc) {
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5, q = lane % C::L;
    F2 rate[C::N / 2];
    const float scale = *dloss;
#pragma unroll
    for (int i = 0; i < C::N / 2; ++i) {
        float r[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int at = 2 * i + k, e = (C::L * (at / C::V) + q) * C::V + at % C::V;
            r[k] = e < p.experts ? rates[e] : 0.0f;
        }
        rate[i] = F2(r[0], r[1]);
    }
    constexpr int ES = C::T == GK_F32 ? 4 : 2;
    const int64_t step = static_cast<int64_t>(gridDim.x) * warps * C::G * C::U;
    for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * warps + w) * C::G * C::U; t0 < p.tokens; t0 += step) {
        Logits<C> x[C::U];
#pragma unroll
        for (int k = 0; k < C::U; ++k) {
            const int64_t t = t0 + k * C::G + lane / C::L;
            if (t < p.tokens) x[k].load(p, t, q);
        }
#pragma unroll
        for (int k = 0; k < C::U; ++k) {
            const int64_t t = t0 + k * C::G + lane / C::L;
            const bool has = token_ids<C::L>(p, t, t < p.tokens, nullptr, lane);
            F2 y[C::N / 2];
            const float inv = x[k].softmax(p, q, y);
            F2 dot2(0.0f);
#pragma unroll
            for (int i = 0; i < C::N / 2; ++i) dot2 = fma2(y[i], rate[i], dot2);
            float dot = dot2.lo() + dot2.hi();
#pragma unroll
            for (int d = C::L / 2; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
            const F2 less(-(dot * inv)), f(scale * inv);
#pragma unroll
            for (int i = 0; i < C::N / 2; ++i)  // (padding may hold anything)
                y[i] = has ? mul2(mul2(y[i], f), add2(rate[i], less)) : F2(0.0f);
            if (t >= p.tokens) continue;
            uint8_t* row = static_cast<uint8_t*>(dx) + (t * ds + (C::V == 4 ? q * C::V : 0)) * ES;
#pragma unroll
            for (int j = 0; j < C::J; ++j) {
                const int e = (C::L * j + q) * C::V;
                if (e >= p.experts) continue;
                if constexpr (C::V == 1) {
                    const float g = j & 1 ? y[j / 2].hi() : y[j / 2].lo();
                    uint8_t* at = row + e * dc * ES;
                    if (C::T == GK_F32)
                        to_out(reinterpret_cast<float*>(at), g);
                    else if (C::T == GK_F16)
                        to_out(reinterpret_cast<__half*>(at), g);
                    else
                        to_out(reinterpret_cast<__nv_bfloat16*>(at), g);
                } else {
                    uint8_t* at = row + C::L * j * C::V * ES;
                    uint32_t b[4];
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        const F2 pair = y[(4 * j + v) / 2];
                        b[v] = __float_as_uint(v & 1 ? pair.hi() : pair.lo());
                    }
                    if (C::T == GK_F32)
                        st_global_v4(at, b[0], b[1], b[2], b[3]);
                    else
                        *reinterpret_cast<uint2*>(at) = make_uint2(round_pair(b[0], b[1], 1.0f, C::T),
                                                                   round_pair(b[2], b[3], 1.0f, C::T));
                }
            }
        }
    }
}

// f(a Layout): V = 4 where a row's logits are whole 4-element pieces, sixteen logits a lane where the
// experts allow that (fewer lanes a token mean fewer steps over lanes), 32 at most.
template <typename F>
int with_layout(int type, bool vec, int experts, F f) {
    auto pick = [&](auto t) {
        constexpr int T = decltype(t)::value;
        if (vec) {
            if (experts <= 16) return f(Layout<T, 4, 4, 1>{});
            if (experts <= 64) return f(Layout<T, 4, 4, 4>{});
            if (experts <= 256) return f(Layout<T, 4, 4, 16>{});
            if (experts <= 512) return f(Layout<T, 4, 4, 32>{});
            return f(Layout<T, 4, 8, 32>{});
        }
        if (experts <= 64) return f(Layout<T, 1, 16, 4>{});
        if (experts <= 256) return f(Layout<T, 1, 16, 16>{});
        if (experts <= 512) return f(Layout<T, 1, 16, 32>{});
        return f(Layout<T, 1, 32, 32>{});
    };
    if (type == GK_F32) return pick(std::integral_constant<int, GK_F32>{});
    if (type == GK_F16) return pick(std::integral_constant<int, GK_F16>{});
    return pick(std::integral_constant<int, GK_BF16>{});
}

// Tokens of a warp at a time.
int tokens_a_step(int type, bool vec, int experts) {
    return with_layout(type, vec, experts, [](auto layout) {
        using C = decltype(layout);
        return C::G * C::U;
    });
}

bool in_fours(const void* p, int64_t rows, int64_t cols, int64_t rs, int64_t cs, size_t es) {
    return cs == 1 && cols % 4 == 0 && (rows <= 1 || rs % 4 == 0) &&
           reinterpret_cast<uintptr_t>(p) % (4 * es) == 0;
}

size_t view_bytes(size_t rows, size_t cols, ptrdiff_t rs, ptrdiff_t cs, size_t es) {
    return rows && cols ? ((rows - 1) * rs + (cols - 1) * cs + 1) * es : 0;
}

int check_router(const gk_matref& x, int x_type, const void* ids, size_t ids_len, size_t top, int ids64,
                 Router* p) {
    if (x_type != GK_F32 && x_type != GK_F16 && x_type != GK_BF16)
        return api_err(GK_EINVAL, "gemmkit: unknown element type %d", x_type);
    int rc = api_check_view(x.len, x.rows, x.cols, x.rs, x.cs, "logits");
    if (rc) return rc;
    if (x.cols < 1 || x.cols > MAX_EXPERTS)
        return api_err(GK_EINVAL, "gemmkit: a router has 1 to %d experts (has %zu)", MAX_EXPERTS, x.cols);
    if (top < 1 || top > INT32_MAX / 2 || x.rows > INT32_MAX / 2 || x.rows * top > INT32_MAX)
        return api_err(GK_EINVAL, "gemmkit: problem dimensions exceed the engine's limits");
    if (ids_len < x.rows * top)
        return api_err(GK_EINVAL, "gemmkit: %zu tokens with %zu experts each need as many ids (has %zu)",
                       x.rows, top, ids_len);
    if (x.rows && (!x.data || !ids)) return api_err(GK_EINVAL, "gemmkit: null logits or ids");
    if ((rc = api_check_aligned(x.data, x_type == GK_F32 ? 4 : 2, "logits")) ||
        (rc = api_check_aligned(ids, ids64 ? 8 : 4, "ids")))
        return rc;
    *p = Router{x.data, x.rs, x.cs, ids64 != 0, ids, static_cast<int32_t>(top),
                static_cast<int32_t>(x.rows), static_cast<int32_t>(x.cols), nullptr};
    return GK_OK;
}

}  // namespace

}  // namespace gk

using namespace gk;

extern "C" {

int gk_moe_balance(gk_matref logits, int x_type, const void* ids, size_t ids_len, size_t top, int ids64,
                   float coef, float* loss, int32_t* counts, int32_t* offsets, float* rates,
                   gk_stream_t stream) {
    Router p;
    int rc = check_router(logits, x_type, ids, ids_len, top, ids64, &p);
    if (rc) return rc;
    if (!loss || !counts || !offsets || !rates) return api_err(GK_EINVAL, "gemmkit: null output");
    if ((rc = api_check_aligned(loss, 4, "loss")) || (rc = api_check_aligned(counts, 4, "counts")) ||
        (rc = api_check_aligned(offsets, 4, "offsets")) || (rc = api_check_aligned(rates, 4, "rates")))
        return rc;
    const size_t es = x_type == GK_F32 ? 4 : 2, n = logits.cols;
    const struct {
        const void* p;
        size_t bytes;
    } all[6] = {{loss, 4},  {counts, 4 * n}, {offsets, 4 * (n + 1)},
                {rates, 4 * n},
                {logits.data, view_bytes(logits.rows, n, logits.rs, logits.cs, es)},
                {ids, logits.rows * top * (ids64 ? 8 : 4)}};
    for (int i = 0; i < 4; ++i)
        for (int j = i + 1; j < 6; ++j)
            if (all[j].p && all[j].bytes && api_overlaps(all[i].p, all[i].bytes, all[j].p, all[j].bytes))
                return api_err(GK_EINVAL, "gemmkit: the outputs alias each other or the inputs");
    int dev = 0;
    if ((rc = api_check_device(&dev))) return rc;
    p.status = device_status_ptr();
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool vec = in_fours(logits.data, p.tokens, p.experts, p.rs, p.cs, es);
    // a block more for each step of tokens, up to what is resident
    const int64_t step = BW * tokens_a_step(x_type, vec, p.experts), most = 2ll * sm_count();
    const int64_t want = (p.tokens + step - 1) / step;
    const int blocks = static_cast<int>(want < 1 ? 1 : want < most ? want : most);
    const BalanceOut o{coef, loss, counts, offsets, rates};
    void* part = nullptr;
    if (blocks > 1 &&
        (rc = scratch_alloc(&part, static_cast<size_t>(part_words(blocks, p.experts)) * 4, st)))
        return rc;
    rc = with_layout(x_type, vec, p.experts, [&](auto layout) {
        using C = decltype(layout);
        auto kern = balance_kernel<C>;
        const int smem = ((BW + 2) * p.experts + 1) * 4;
        static std::atomic<uint64_t> done{0};
        const cudaError_t e = allow_smem(kern, ((BW + 2) * MAX_EXPERTS + 1) * 4, done);
        if (e != cudaSuccess)
            return api_err(GK_ECUDA, "gemmkit: kernel launch failed: %s", cudaGetErrorString(e));
        return launch_overlapped_smem(kern, dim3(static_cast<unsigned>(blocks)), 32 * BW, smem, st, p,
                                      static_cast<uint32_t*>(part), o);
    });
    if (!rc && blocks > 1)
        rc = launch_overlapped(balance_finish_kernel, dim3(static_cast<unsigned>((p.experts + 31) / 32)),
                               32 * FW, st, static_cast<uint32_t*>(part), blocks, p.experts, o);
    const int fr = scratch_free(part, st);
    return rc ? rc : fr;
}

int gk_moe_balance_backward(gk_matref logits, int x_type, const void* ids, size_t ids_len, size_t top,
                            int ids64, const float* rates, const float* dloss, gk_matmut dlogits,
                            gk_stream_t stream) {
    Router p;
    int rc = check_router(logits, x_type, ids, ids_len, top, ids64, &p);
    if (rc) return rc;
    if (dlogits.rows != logits.rows || dlogits.cols != logits.cols)
        return api_err(GK_EINVAL, "gemmkit: the gradient is %zux%zu, the logits are %zux%zu", dlogits.rows,
                       dlogits.cols, logits.rows, logits.cols);
    if ((rc = api_check_view(dlogits.len, dlogits.rows, dlogits.cols, dlogits.rs, dlogits.cs, "dlogits")))
        return rc;
    if (api_self_aliases(dlogits.rows, dlogits.cols, dlogits.rs, dlogits.cs))
        return api_err(GK_EINVAL, "gemmkit: dlogits view aliases itself");
    if (!rates || !dloss) return api_err(GK_EINVAL, "gemmkit: null rates or dloss");
    if (p.tokens == 0) return GK_OK;
    if (!dlogits.data) return api_err(GK_EINVAL, "gemmkit: null dlogits");
    const size_t es = x_type == GK_F32 ? 4 : 2, n = logits.cols;
    if ((rc = api_check_aligned(dlogits.data, es, "dlogits")) ||
        (rc = api_check_aligned(rates, 4, "rates")) || (rc = api_check_aligned(dloss, 4, "dloss")))
        return rc;
    const size_t db = view_bytes(dlogits.rows, n, dlogits.rs, dlogits.cs, es);
    const bool same = dlogits.data == logits.data && (p.tokens <= 1 || dlogits.rs == logits.rs) &&
                      (n <= 1 || dlogits.cs == logits.cs);
    if ((!same && api_overlaps(dlogits.data, db, logits.data,
                               view_bytes(logits.rows, n, logits.rs, logits.cs, es))) ||
        api_overlaps(dlogits.data, db, ids, logits.rows * top * (ids64 ? 8 : 4)) ||
        api_overlaps(dlogits.data, db, rates, 4 * n) || api_overlaps(dlogits.data, db, dloss, 4))
        return api_err(GK_EINVAL, "gemmkit: dlogits alias another operand");
    int dev = 0;
    if ((rc = api_check_device(&dev))) return rc;
    p.status = device_status_ptr();
    const bool vec = in_fours(logits.data, p.tokens, p.experts, p.rs, p.cs, es) &&
                     in_fours(dlogits.data, p.tokens, p.experts, dlogits.rs, dlogits.cs, es);
    const int64_t step = 8 * tokens_a_step(x_type, vec, p.experts), most = 4ll * sm_count();
    const int64_t want = (p.tokens + step - 1) / step;
    return with_layout(x_type, vec, p.experts, [&](auto layout) {
        using C = decltype(layout);
        return launch_overlapped(balance_backward_kernel<C>,
                                 dim3(static_cast<unsigned>(want < most ? want : most)), 256,
                                 static_cast<cudaStream_t>(stream), p, rates, dloss, dlogits.data,
                                 static_cast<int64_t>(dlogits.rs), static_cast<int64_t>(dlogits.cs));
    });
}

}  // extern "C"
