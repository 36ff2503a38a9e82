// gk_grouped.cu -- the products of rows grouped by expert (gk_grouped.cuh): the C entries, the copies of
// operands that TMA cannot address, and the engine's stream-ordered scratch memory.
#include <mutex>

#include "gk_grouped.cuh"

namespace gk {

namespace {

// ---- operands that TMA cannot address --------------------------------------------------------------
// (Plain loads: these kernels may start before the kernel that writes their source has ended, and
// only wait for it, so the source is not read-only for their lifetime.)

// The 16 bytes at byte offset a (0, 2 .. 14) of the 32 in (lo, hi).
__device__ __forceinline__ uint4 shift_bytes(const uint4& lo, const uint4& hi, uint32_t a) {
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (a & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (a & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const uint32_t b = (a & 2) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], b), __funnelshift_r(w[1], w[2], b),
                      __funnelshift_r(w[2], w[3], b), __funnelshift_r(w[3], w[4], b));
}

constexpr int RU = 4;  // 16-byte pieces of a lane in flight

// dst[g][l][e] = src[g * gs + l * pitch + e] for l < lines, e < len, zero for len <= e < dld (dld a
// multiple of 8): lines that start at any 2-byte address, to 16-byte aligned ones. A warp takes
// RU * 256 elements of a line; a piece is two aligned 16-byte loads shifted together (one where
// the line is aligned), or single elements where those would leave the source's bytes [lo, hi).
__global__ void __launch_bounds__(256)
    realign_lines_kernel(uint16_t* dst, int64_t dld, const uint16_t* src,
                         int64_t pitch, int64_t gs, int64_t lines, int64_t len, int64_t groups,
                         const uint8_t* lo, const uint8_t* hi) {
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t chunks = (dld + RU * 256 - 1) / (RU * 256);
    const int64_t units = groups * lines * chunks;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
         u < units; u += step) {
        const int64_t gl = u / chunks, c = u - gl * chunks;
        const int64_t g = gl / lines, l = gl - g * lines;
        const uint16_t* s = src + g * gs + l * pitch;
        uint16_t* d = dst + gl * dld;
        const int64_t e0 = c * (RU * 256) + lane * 8;
        const uint32_t a = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(s)) & 15u;
        uint4 x[RU], y[RU];
#pragma unroll
        for (int i = 0; i < RU; ++i) {
            const int64_t e = e0 + i * 256;
            const int n = static_cast<int>(min(static_cast<int64_t>(8), len - e));
            x[i] = y[i] = make_uint4(0, 0, 0, 0);
            if (n <= 0) continue;
            const uint8_t* p = reinterpret_cast<const uint8_t*>(s + e) - a;
            const bool two = a + 2 * n > 16;
            if (p >= lo && p + (two ? 32 : 16) <= hi) {
                x[i] = *reinterpret_cast<const uint4*>(p);
                if (two) y[i] = reinterpret_cast<const uint4*>(p)[1];
            } else {  // placed so that the shift below finds them
                uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (k < n) {
                        const uint32_t at = a / 2 + k;
                        const uint32_t v = static_cast<uint32_t>(s[e + k]) << (16 * (at & 1));
#pragma unroll
                        for (uint32_t q = 0; q < 8; ++q)
                            if ((at >> 1) == q) w[q] |= v;
                    }
                x[i] = make_uint4(w[0], w[1], w[2], w[3]);
                y[i] = make_uint4(w[4], w[5], w[6], w[7]);
            }
        }
#pragma unroll
        for (int i = 0; i < RU; ++i) {
            const int64_t e = e0 + i * 256;
            if (e >= dld) break;
            uint4 q = shift_bytes(x[i], y[i], a);
            const int64_t n = len - e;
            q.x = n > 1 ? q.x : n > 0 ? q.x & 0xFFFFu : 0u;
            q.y = n > 3 ? q.y : n > 2 ? q.y & 0xFFFFu : 0u;
            q.z = n > 5 ? q.z : n > 4 ? q.z & 0xFFFFu : 0u;
            q.w = n > 7 ? q.w : n > 6 ? q.w & 0xFFFFu : 0u;
            *reinterpret_cast<uint4*>(d + e) = q;
        }
    }
}

// dst[g][l][e] = src[g * gs + l * sl + e * se], padded likewise, through a 32 x 32 tile: both sides
// are coalesced whichever source stride is small.
__global__ void __launch_bounds__(256)
    realign_any_kernel(uint16_t* dst, int64_t dld, const uint16_t* src,
                       int64_t sl, int64_t se, int64_t gs, int64_t lines, int64_t len,
                       int64_t groups) {
    __shared__ uint16_t tile[32][33];
    griddep_wait();
    griddep_launch_dependents();
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t te = (dld + 31) / 32, tl = (lines + 31) / 32;
    const bool e_fast = se <= sl;
    for (int64_t t = blockIdx.x; t < groups * tl * te; t += gridDim.x) {
        const int64_t g = t / (tl * te), r = t - g * tl * te;
        const int64_t l0 = r / te * 32, e0 = (r - r / te * te) * 32;
        for (int i = ty; i < 32; i += 8) {
            const int64_t l = l0 + (e_fast ? i : tx), e = e0 + (e_fast ? tx : i);
            const uint16_t v =
                l < lines && e < len ? src[g * gs + l * sl + e * se] : uint16_t{0};
            tile[e_fast ? i : tx][e_fast ? tx : i] = v;
        }
        __syncthreads();
        for (int i = ty; i < 32; i += 8) {
            const int64_t l = l0 + i, e = e0 + tx;
            if (l < lines && e < dld) dst[(g * lines + l) * dld + e] = tile[i][tx];
        }
        __syncthreads();
    }
}

// Scratch for realigned operands: stream-ordered memory from a pool of the engine's own on the
// current device, so that calls on several streams, and calls captured into several graphs, never
// share any (a captured call allocates and frees inside its graph). At every synchronisation the
// pool gives back what it holds beyond 1 / SCRATCH_SHARE of the device's memory (2.8 of 179 GiB), and
// gk_scratch_release the rest. (Held without a bound, one call with a large stack of odd weights
// kept its size from the process's other allocations for good. Mapping memory anew is not cheap:
// with a bound below its 0.94 GB a synchronised call with 8 weights of 4096 x 14336 took 2.3
// instead of 0.49 ms.)
constexpr size_t SCRATCH_SHARE = 64;

// The pool of device `dev`; with `make`, made at the first call (nullptr on failure).
cudaMemPool_t scratch_pool(int dev, bool make) {
    static std::mutex m;
    static cudaMemPool_t pools[64] = {};
    if (dev < 0 || dev >= 64) return nullptr;
    std::lock_guard<std::mutex> lock(m);
    if (!pools[dev] && make) {
        cudaMemPoolProps props;
        memset(&props, 0, sizeof(props));
        props.allocType = cudaMemAllocationTypePinned;
        props.handleTypes = cudaMemHandleTypeNone;
        props.location.type = cudaMemLocationTypeDevice;
        props.location.id = dev;
        size_t unused = 0, total = 0;
        cudaMemPool_t pool = nullptr;
        if (cudaMemGetInfo(&unused, &total) != cudaSuccess ||
            cudaMemPoolCreate(&pool, &props) != cudaSuccess) {
            cudaGetLastError();
            return nullptr;
        }
        uint64_t keep = total / SCRATCH_SHARE;
        if (cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep) != cudaSuccess)
            cudaGetLastError();  // it then keeps nothing
        pools[dev] = pool;
    }
    return pools[dev];
}

}  // namespace

// `bytes` of scratch for calls on `st`; freed by scratch_free on the same stream.
int scratch_alloc(void** scratch, size_t bytes, cudaStream_t st) {
    // a captured allocation belongs to its graph, whichever pool it names (and a pool cannot be
    // created during a capture)
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamIsCapturing(st, &cap);
    if (e == cudaSuccess && cap != cudaStreamCaptureStatusNone) {
        e = cudaMallocAsync(scratch, bytes, st);
    } else if (e == cudaSuccess) {
        int dev = -1;
        cudaGetDevice(&dev);
        cudaMemPool_t pool = scratch_pool(dev, true);
        e = pool ? cudaMallocFromPoolAsync(scratch, bytes, pool, st) : cudaErrorMemoryAllocation;
        if (e == cudaErrorMemoryAllocation && pool) {  // once more, without what the pool holds unused
            cudaGetLastError();
            cudaMemPoolTrimTo(pool, 0);
            e = cudaMallocFromPoolAsync(scratch, bytes, pool, st);
        }
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        *scratch = nullptr;
        return api_err(e == cudaErrorMemoryAllocation ? GK_ENOMEM : GK_ECUDA,
                       "gemmkit: workspace allocation: %s", cudaGetErrorString(e));
    }
    return GK_OK;
}

int scratch_free(void* scratch, cudaStream_t st) {
    if (scratch && cudaFreeAsync(scratch, st) != cudaSuccess) {
        cudaGetLastError();
        return api_err(GK_ECUDA, "gemmkit: freeing the workspace failed");
    }
    return GK_OK;
}

int realign(GOperand* o, int64_t rows, int64_t len, int64_t groups, bool mn, int pdl,
            cudaStream_t st, void** scratch) {
    const int64_t lines = mn ? len : rows, run = mn ? rows : len;
    const int64_t sl = mn ? o->ps : o->rs, se = mn ? o->rs : o->ps;
    const int64_t dld = (run + 7) / 8 * 8;
    if (int rc = scratch_alloc(scratch, static_cast<size_t>(groups * lines * dld * 2), st)) return rc;
    cudaError_t e;
    uint16_t* dst = static_cast<uint16_t*>(*scratch);
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    const int64_t most = static_cast<int64_t>(sm_count()) * 8;
    if (se == 1 || run <= 1) {
        const int64_t units = groups * lines * ((dld + RU * 256 - 1) / (RU * 256));
        const int64_t blocks = (units + 7) / 8;
        cfg.gridDim = dim3(static_cast<unsigned>(blocks < most ? blocks : most));
        const uint8_t* lo = reinterpret_cast<const uint8_t*>(o->ptr);
        const uint8_t* hi = reinterpret_cast<const uint8_t*>(
            o->ptr + (groups - 1) * o->gs + (lines - 1) * sl + run);
        e = cudaLaunchKernelEx(&cfg, realign_lines_kernel, dst, dld, o->ptr, sl, o->gs, lines, run,
                               groups, lo, hi);
    } else {
        const int64_t tiles = groups * ((lines + 31) / 32) * ((dld + 31) / 32);
        cfg.gridDim = dim3(static_cast<unsigned>(tiles < most ? tiles : most));
        e = cudaLaunchKernelEx(&cfg, realign_any_kernel, dst, dld, o->ptr, sl, se, o->gs, lines, run,
                               groups);
    }
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess)
        return api_err(GK_ECUDA, "gemmkit: pack kernel launch failed: %s", cudaGetErrorString(e));
    *o = mn ? GOperand{dst, 1, dld, lines * dld} : GOperand{dst, dld, 1, lines * dld};
    return GK_OK;
}

// The weight gradient's checks; `held`: A is held in another form (its address is not looked at), and
// offsets may be missing, for one group of all rows.
int check_wgrad(int is_f16, size_t groups, const int32_t* offsets, bool held, float alpha,
                const gk_matref& a, const gk_matref& b, const gk_matmut& c, ptrdiff_t c_gs,
                int out_type) {
    static const int32_t all = 0;
    int rc = check_groups(groups, held && groups == 1 && !offsets ? &all : offsets, a.rows, is_f16,
                          out_type);
    if (rc) return rc;
    const size_t so = out_type == GK_F32 ? 4 : 2;
    // A^T B in gemmkit's frame: (A.cols x rows) (rows x B.cols)
    const gk_matref at{a.data, a.len, a.cols, a.rows, a.cs, a.rs};
    if ((rc = api_validate_gemm_views(at, b, c, 2, so))) return rc;
    const gk_matref cr{c.data, c.len, c.rows, c.cols, c.rs, c.cs};
    if ((rc = check_stack(cr.len, groups, cr.rows, cr.cols, cr.rs, cr.cs, c_gs, "C"))) return rc;
    if (a.cols > INT32_MAX / 2 || b.cols > INT32_MAX / 2)
        return api_err(GK_EINVAL, "gemmkit: problem dimensions exceed the engine's limits");
    if (c.rows == 0 || c.cols == 0) return GK_OK;
    if (groups > 1) {  // no element of one group's C may be an element of another's
        size_t need = static_cast<size_t>((c.rows - 1) * c.rs + (c.cols - 1) * c.cs) + 1;
        if (static_cast<size_t>(c_gs) < need)
            return api_err(GK_EINVAL,
                           "gemmkit: the groups of C overlap or interleave (group stride %td, a group "
                           "spans %zu elements)",
                           c_gs, need);
    }
    if (!c.data) return api_err(GK_EINVAL, "gemmkit: null C");
    const bool zero = a.rows == 0 || alpha == 0.0f;
    if (!zero && ((!held && !a.data) || !b.data)) return api_err(GK_EINVAL, "gemmkit: null A or B");
    if ((rc = api_check_aligned(a.data, 2, "A")) || (rc = api_check_aligned(b.data, 2, "B")) ||
        (rc = api_check_aligned(c.data, so, "C")))
        return rc;
    return GK_OK;
}

// The weight gradient, its arguments checked; offsets == nullptr: one group of all rows.
int run_wgrad(int is_f16, size_t groups, const int32_t* offsets, float alpha, const gk_matref& a,
              const gk_matref& b, float beta, const gk_matmut& c, ptrdiff_t c_gs, int out_type,
              cudaStream_t stream) {
    GroupedParams p;
    memset(&p, 0, sizeof(p));
    p.P = GOperand{static_cast<const uint16_t*>(b.data), b.cs, b.rs, 0};
    p.Q = GOperand{static_cast<const uint16_t*>(a.data), a.cs, a.rs, 0};
    p.np = static_cast<int64_t>(b.cols);
    p.nq = static_cast<int64_t>(a.cols);
    p.wgrad = 1;
    p.zero = a.rows == 0 || alpha == 0.0f;
    p.groups = static_cast<int>(groups);
    p.rows = static_cast<int>(a.rows);
    p.offsets = offsets;
    p.c = c.data;
    p.ldq = c.rs;
    p.ldp = c.cs;
    p.gsc = c_gs;
    p.alpha = alpha;
    p.beta = beta;
    p.f16 = is_f16 != 0;
    p.out_type = out_type;
    return run_grouped<EPI_STORE>(p, stream);
}

}  // namespace gk

using namespace gk;

extern "C" {

int gk_scratch_release(int device) {
    int prev = 0;
    cudaGetDevice(&prev);
    if (cudaSetDevice(device) != cudaSuccess) {
        cudaGetLastError();
        return api_err(GK_ENODEV, "gemmkit: bad device");
    }
    cudaMemPool_t pool = scratch_pool(device, false);
    cudaError_t e = cudaSuccess;
    if (pool) {  // what was freed is unused once the calls that used it have ended
        e = cudaDeviceSynchronize();
        if (e == cudaSuccess) e = cudaMemPoolTrimTo(pool, 0);
    }
    cudaSetDevice(prev);
    if (e != cudaSuccess)
        return api_err(GK_ECUDA, "gemmkit: releasing the scratch: %s", cudaGetErrorString(e));
    return GK_OK;
}

int gk_gemm_half_grouped(int is_f16, size_t groups, const int32_t* offsets, float alpha,
                         gk_matref a, gk_matref b, ptrdiff_t b_gs, float beta, gk_matmut c,
                         int out_type, gk_parallelism par, gk_stream_t stream) {
    (void)par;
    int rc = check_groups(groups, offsets, a.rows, is_f16, out_type);
    if (rc) return rc;
    const size_t so = out_type == GK_F32 ? 4 : 2;
    if ((rc = api_validate_gemm_views(a, b, c, 2, so))) return rc;
    if ((rc = check_stack(b.len, groups, b.rows, b.cols, b.rs, b.cs, b_gs, "B"))) return rc;
    if (a.cols > INT32_MAX / 2 || b.cols > INT32_MAX / 2)
        return api_err(GK_EINVAL, "gemmkit: problem dimensions exceed the engine's limits");
    if (c.rows == 0 || c.cols == 0) return GK_OK;
    if (!c.data) return api_err(GK_EINVAL, "gemmkit: null C");
    const bool zero = a.cols == 0 || alpha == 0.0f;
    if (!zero && (!a.data || !b.data)) return api_err(GK_EINVAL, "gemmkit: null A or B");
    if ((rc = api_check_aligned(a.data, 2, "A")) || (rc = api_check_aligned(b.data, 2, "B")) ||
        (rc = api_check_aligned(c.data, so, "C")))
        return rc;
    GroupedParams p;
    memset(&p, 0, sizeof(p));
    p.P = GOperand{static_cast<const uint16_t*>(b.data), b.cs, b.rs, b_gs};
    p.Q = GOperand{static_cast<const uint16_t*>(a.data), a.rs, a.cs, 0};
    p.np = static_cast<int64_t>(b.cols);
    p.kdim = static_cast<int32_t>(a.cols);
    p.zero = zero;
    p.groups = static_cast<int>(groups);
    p.rows = static_cast<int>(a.rows);
    p.offsets = offsets;
    p.c = c.data;
    p.ldq = c.rs;
    p.ldp = c.cs;
    p.alpha = alpha;
    p.beta = beta;
    p.f16 = is_f16 != 0;
    p.out_type = out_type;
    return run_grouped<EPI_STORE>(p, static_cast<cudaStream_t>(stream));
}

int gk_gemm_half_grouped_wgrad(int is_f16, size_t groups, const int32_t* offsets, float alpha,
                               gk_matref a, gk_matref b, float beta, gk_matmut c, ptrdiff_t c_gs,
                               int out_type, gk_parallelism par, gk_stream_t stream) {
    (void)par;
    int rc = check_wgrad(is_f16, groups, offsets, false, alpha, a, b, c, c_gs, out_type);
    if (rc || c.rows == 0 || c.cols == 0) return rc;
    return run_wgrad(is_f16, groups, offsets, alpha, a, b, beta, c, c_gs, out_type,
                     static_cast<cudaStream_t>(stream));
}

}  // extern "C"
