// gk_linear.cu -- a feed-forward layer's products with their epilogues, and their backward pass
// (gk_grouped.cuh with the epilogues of gk_epilogue.cuh):
//
//   forward         z = alpha A B[g] + bias[g];  C = act(z) + R
//   input gradient  C = alpha A B[g] * act'(z);  dbias[g] = sums of C over the group's rows
//   without a product                dz = dy * act'(z);  dbias[g] likewise
#include "gk_grouped.cuh"
#include "gk_launch.h"

namespace gk {

namespace {

// ---- column sums ----------------------------------------------------------------------------------------
//
// Whoever computes the gradient leaves the sums of its parts of a group in consecutive slots of np f32: the
// tiles of `tile` rows of a group, `shares` slots each; or, with `slice`, the pieces of slices of that many
// rows that lie in the group, slice s of group g in slot s + g (two pieces that meet in a slice or in a
// group never share one). No atomics, so the sums repeat bit for bit. A warp of the second kernel takes
// 32 columns of a group and adds an eighth of the slots in f64.

constexpr int SUM_WARPS = 8;

__global__ void __launch_bounds__(32 * SUM_WARPS)
    sum_parts_kernel(const float* part, const int32_t* offsets, int groups, int rows, int tile,
                     int shares, int slice, int64_t np, void* out, int64_t gs, int type) {
    __shared__ int off[GROUP_TABLE_INTS], tile0[GROUP_TABLE_INTS];
    __shared__ double s[SUM_WARPS][32];
    griddep_wait();
    griddep_launch_dependents();
    load_groups(offsets, groups, rows, off, tile0, nullptr,
                [&](int m) { return slice ? 0 : (m + tile - 1) / tile; });
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = blockIdx.y;
    int64_t first = static_cast<int64_t>(tile0[g]) * shares,
            end = static_cast<int64_t>(tile0[g + 1]) * shares;
    if (slice && off[g] < off[g + 1]) {
        first = off[g] / slice + g;
        end = (off[g + 1] - 1) / slice + g + 1;
    }
    const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    double a = 0.0;
    if (col < np) {
#pragma unroll 4
        for (int64_t i = first + w; i < end; i += SUM_WARPS)
            a += static_cast<double>(part[i * np + col]);
    }
    s[w][lane] = a;
    __syncthreads();
    if (w != 0 || col >= np) return;
#pragma unroll
    for (int i = 1; i < SUM_WARPS; ++i) a += s[i][lane];
    const float y = static_cast<float>(a);
    const int64_t at = g * gs + col;
    if (type == GK_F32)
        to_out(static_cast<float*>(out) + at, y);
    else if (type == GK_F16)
        to_out(static_cast<__half*>(out) + at, y);
    else
        to_out(static_cast<__nv_bfloat16*>(out) + at, y);
}

}  // namespace

int launch_sum_parts(const float* part, const int32_t* offsets, int groups, int rows, int tile,
                     int shares, int slice, int64_t np, const EpiArgs& e, cudaStream_t st) {
    const dim3 grid(static_cast<unsigned>((np + 31) / 32), static_cast<unsigned>(groups));
    return launch_overlapped(sum_parts_kernel, grid, 32 * SUM_WARPS, st, part, offsets, groups, rows,
                             tile, shares, slice, np, e.dbias, e.dbias_gs, e.bias_type);
}

namespace {

// ---- the gradient without a product -----------------------------------------------------------------------
//
// Bound by memory: dy and z are read and dz is written once. The rows are cut into as many equal slices as
// make the grid what is resident; a block walks one slice's 32 V columns, group by group, a warp every
// eighth row, with V consecutive columns a lane (16 bytes) where every matrix allows that, else one. Rows
// are read four at a time so that enough loads are in flight. A block's sums stay in registers to the end of a group. (Tiles of 64
// rows, their sums added in shared memory after each: 49 to 65 us for 8192 x 4096 by 8 groups with
// SiLU, now 35.)

constexpr int GW = 8, GU = 4;  // warps, rows of a warp at a time

struct ActGrad {
    const uint16_t* dy;
    int64_t yq, yp;       // strides along rows and columns
    void* dz;             // nullptr: only the sums
    int64_t zq, zp;
    int64_t np;
    const int32_t* offsets;
    int groups, rows, f16, out_type;
    int slice;            // rows of a block
    float* part;
    unsigned int* status;
    EpiArgs e;
};

// V consecutive values of one row: 16 bits, or 8-bit codes and their exponent byte.
template <int V>
struct GradRow {
    uint32_t y[(V + 1) / 2], z[(V + 1) / 2], x;
    __device__ __forceinline__ static void pieces(uint32_t (&w)[(V + 1) / 2], const uint8_t* p) {
        if constexpr (V == 8) {
            const uint4 a = ld_global_v4(p);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        }
    }
    __device__ __forceinline__ void codes(const uint8_t* p) {
        if constexpr (V == 8) {
            const uint2 a = *reinterpret_cast<const uint2*>(p);
            z[0] = a.x, z[1] = a.y;
        } else {
            z[0] = *p;
        }
    }
};

// ACT: the activation, or -1 for the one that p names.
template <int V, bool F16, int ACT>
__global__ void __launch_bounds__(32 * GW, 3) act_grad_kernel(const ActGrad p) {
    constexpr int W = (V + 1) / 2;
    __shared__ int off[GROUP_TABLE_INTS], unused[GROUP_TABLE_INTS];
    __shared__ float red[GW][32 * V];
    griddep_wait();
    griddep_launch_dependents();
    load_groups(p.offsets, p.groups, p.rows, off, unused, blockIdx.x == 0 ? p.status : nullptr,
                [](int) { return 0; });
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const unsigned blocks = static_cast<unsigned>((p.np + 32 * V - 1) / (32 * V));  // along the columns
    const int s = static_cast<int>(blockIdx.x / blocks);
    const int64_t c0 = static_cast<int64_t>(blockIdx.x % blocks) * 32 * V, c = c0 + lane * V;
    const int s0 = s * p.slice, s1 = min(s0 + p.slice, p.rows);
    int g = 0, hi = p.groups;  // the first group that ends behind the slice's first row
    while (g < hi) {
        const int mid = (g + hi) >> 1;
        if (off[mid + 1] > s0)
            hi = mid;
        else
            g = mid + 1;
    }
    const int osize = p.out_type == GK_F32 ? 4 : 2;
    const bool z8 = p.e.z8.codes != nullptr;
    const int64_t ystep = p.yq * 2 * GW, ostep = p.zq * osize * GW, xstep = p.e.z8.exps_ld * GW,
                  zstep = (z8 ? p.e.z8.codes_ld : p.e.sq * 2) * GW;
    for (; g < p.groups && off[g] < s1; ++g) {
        const int r0 = max(off[g], s0), r1 = min(off[g + 1], s1);
        if (r0 >= r1) continue;
        // this lane's place in its first row
        const int64_t r = r0 + w;
        const uint8_t* yp = reinterpret_cast<const uint8_t*>(p.dy + r * p.yq + c * p.yp);
        const uint8_t* zp = z8 ? reinterpret_cast<const uint8_t*>(p.e.z8.codes + r * p.e.z8.codes_ld + c)
                               : static_cast<const uint8_t*>(p.e.side) + (r * p.e.sq + c * p.e.sp) * 2;
        const uint8_t* xp = p.e.z8.exps + r * p.e.z8.exps_ld + (c >> 5);
        uint8_t* op = static_cast<uint8_t*>(p.dz) + (r * p.zq + c * p.zp) * osize;
        int left = c < p.np && r0 + w < r1 ? (r1 - r0 - w + GW - 1) / GW : 0;  // rows of this warp
        F2 sum[W];
#pragma unroll
        for (int i = 0; i < W; ++i) sum[i] = F2(0.0f);
#pragma unroll 1
        for (; left > 0; left -= GU) {
            // (no branch between the loads: where a row is missing, the first again)
            GradRow<V> row[GU];
#pragma unroll
            for (int k = 0; k < GU; ++k) GradRow<V>::pieces(row[k].y, yp + (k < left ? k : 0) * ystep);
            if (z8) {
#pragma unroll
                for (int k = 0; k < GU; ++k) {
                    row[k].codes(zp + (k < left ? k : 0) * zstep);
                    row[k].x = xp[(k < left ? k : 0) * xstep];
                }
            } else if (ACT != GK_ACT_NONE && p.e.side) {
#pragma unroll
                for (int k = 0; k < GU; ++k)
                    GradRow<V>::pieces(row[k].z, zp + (k < left ? k : 0) * zstep);
            }
            yp += GU * ystep;
            zp += GU * zstep;
            xp += GU * xstep;
            auto rows = [&](auto in8, auto act) {
                constexpr int A = decltype(act)::value;
#pragma unroll
                for (int k = 0; k < GU; ++k) {
                    if (k >= left) break;
                    F2 d[W];
                    const F2 unit(decltype(in8)::value ? act8_unit(row[k].x) : 0.0f);
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        d[i] = F2(half_lo(row[k].y[i], F16), V == 1 ? 0.0f : half_hi(row[k].y[i], F16));
                        if constexpr (A != GK_ACT_NONE) {
                            F2 z;
                            if constexpr (decltype(in8)::value) {
                                const uint32_t x = row[k].z[i / 2] ^ 0x80808080u;
                                z = mul2(add2(F2(act8_raw(x, 2 * (i & 1)), act8_raw(x, 2 * (i & 1) + 1)),
                                              F2(-8388736.0f)),
                                         unit);
                            } else {
                                z = F2(half_lo(row[k].z[i], F16), half_hi(row[k].z[i], F16));
                            }
                            d[i] = mul2(d[i], act_slope<A>(z, p.e.slope));
                        }
                        sum[i] = add2(sum[i], d[i]);
                    }
                    if (!p.dz) continue;
                    if constexpr (V == 8) {
                        if (p.out_type == GK_F32) {
#pragma unroll
                            for (int i = 0; i < W; i += 2)
                                st_global_v4(op + 8 * i, __float_as_uint(d[i].lo()),
                                             __float_as_uint(d[i].hi()), __float_as_uint(d[i + 1].lo()),
                                             __float_as_uint(d[i + 1].hi()));
                        } else {
                            uint32_t x[W];
#pragma unroll
                            for (int i = 0; i < W; ++i) x[i] = pack_half2(d[i].lo(), d[i].hi(), F16);
                            st_global_v4(op, x[0], x[1], x[2], x[3]);
                        }
                    } else if (p.out_type == GK_F32) {
                        *reinterpret_cast<float*>(op) = d[0].lo();
                    } else {
                        *reinterpret_cast<uint16_t*>(op) =
                            static_cast<uint16_t>(pack_half2(d[0].lo(), 0.0f, F16));
                    }
                    op += ostep;
                }
            };
            auto kinds = [&](auto act) {
                if (z8)
                    rows(std::true_type{}, act);
                else
                    rows(std::false_type{}, act);
            };
            if constexpr (ACT >= 0)
                kinds(std::integral_constant<int, ACT>{});
            else
                with_act(p.e.act, kinds);
        }
        if (!p.part) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) red[w][i * 32 + lane] = i & 1 ? sum[i / 2].hi() : sum[i / 2].lo();
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * V; i += 32 * GW) {  // column (i % 32) V + i / 32 of the block
            float a = red[0][i];
#pragma unroll
            for (int k = 1; k < GW; ++k) a += red[k][i];
            const int64_t col = c0 + (i & 31) * V + (i >> 5);
            if (col < p.np) p.part[static_cast<int64_t>(s + g) * p.np + col] = a;
        }
        __syncthreads();
    }
}

template <bool F16>
void (*act_grad_for(bool vec, int act))(const ActGrad) {
    if (!vec) return act_grad_kernel<1, F16, -1>;
    switch (act) {
        case GK_ACT_RELU: return act_grad_kernel<8, F16, GK_ACT_RELU>;
        case GK_ACT_LEAKY_RELU: return act_grad_kernel<8, F16, GK_ACT_LEAKY_RELU>;
        case GK_ACT_GELU: return act_grad_kernel<8, F16, GK_ACT_GELU>;
        case GK_ACT_GELU_TANH: return act_grad_kernel<8, F16, GK_ACT_GELU_TANH>;
        case GK_ACT_SILU: return act_grad_kernel<8, F16, GK_ACT_SILU>;
        default: return act_grad_kernel<8, F16, GK_ACT_NONE>;
    }
}

// ---- the entries' checks --------------------------------------------------------------------------------

size_t elem_size(int type) { return type == GK_F32 ? 4 : 2; }

// The bytes from a view's first to its last element (0 for an empty one).
size_t span(size_t rows, size_t cols, ptrdiff_t rs, ptrdiff_t cs, size_t es) {
    if (!rows || !cols) return 0;
    return (static_cast<size_t>(rows - 1) * rs + static_cast<size_t>(cols - 1) * cs + 1) * es;
}

struct Span {
    const void* p;
    size_t bytes;
};
Span span_of(const gk_matref& m, size_t es) { return {m.data, span(m.rows, m.cols, m.rs, m.cs, es)}; }
Span span_of(const gk_matmut& m, size_t es) { return {m.data, span(m.rows, m.cols, m.rs, m.cs, es)}; }
bool meet(const Span& a, const Span& b) {
    return a.p && b.p && a.bytes && b.bytes && api_overlaps(a.p, a.bytes, b.p, b.bytes);
}
bool same_view(const gk_matref& a, const gk_matmut& b) {
    return a.data == b.data && (a.rows <= 1 || a.rs == b.rs) && (a.cols <= 1 || a.cs == b.cs);
}

// A matrix of the epilogue: rows x cols like C.
int check_like_c(const gk_matref& m, const gk_matmut& c, size_t es, const char* name) {
    if (m.rows != c.rows || m.cols != c.cols)
        return api_err(GK_EINVAL, "gemmkit: %s is %zux%zu, the output is %zux%zu", name, m.rows, m.cols,
                       c.rows, c.cols);
    int rc = api_check_view(m.len, m.rows, m.cols, m.rs, m.cs, name);
    return rc ? rc : api_check_aligned(m.data, es, name);
}

int check_act(int act) {
    if (act < GK_ACT_NONE || act > GK_ACT_SILU)
        return api_err(GK_EINVAL, "gemmkit: unknown activation %d", act);
    return GK_OK;
}

// n elements a group at stride gs: a bias or its gradient.
int check_vector(const void* p, size_t len, ptrdiff_t gs, int type, size_t groups, size_t n, int is_f16,
                 bool written, const char* name) {
    if (type != GK_F32 && type != (is_f16 ? GK_F16 : GK_BF16))
        return api_err(GK_EINVAL, "gemmkit: %s must hold f32 or the operands' type", name);
    if (gs < 0 || (written && groups > 1 && static_cast<size_t>(gs) < n))
        return api_err(GK_EINVAL, "gemmkit: bad group stride %td of %s", gs, name);
    const unsigned __int128 need = static_cast<unsigned __int128>(groups - 1) * gs + n;
    if (need > len)
        return api_err(GK_EINVAL, "gemmkit: %s holds %zu elements, %zu groups of %zu need %zu", name, len,
                       groups, n, static_cast<size_t>(need));
    return api_check_aligned(p, elem_size(type), name);
}

// What the entries share before their own parts are looked at.
int check_product(int is_f16, size_t groups, const int32_t* offsets, gk_matref a, gk_matref b,
                  ptrdiff_t b_gs, gk_matmut c, int out_type) {
    static const int32_t all = 0;  // stands for the offsets of a plain product
    if (!offsets && groups != 1)
        return api_err(GK_EINVAL, "gemmkit: null offsets");
    int rc = check_groups(groups, offsets ? offsets : &all, a.rows, is_f16, out_type);
    if (rc) return rc;
    if ((rc = api_validate_gemm_views(a, b, c, 2, elem_size(out_type)))) return rc;
    if ((rc = check_stack(b.len, groups, b.rows, b.cols, b.rs, b.cs, b_gs, "B"))) return rc;
    if (a.cols > INT32_MAX / 2 || b.cols > INT32_MAX / 2)
        return api_err(GK_EINVAL, "gemmkit: problem dimensions exceed the engine's limits");
    if ((rc = api_check_aligned(a.data, 2, "A")) || (rc = api_check_aligned(b.data, 2, "B")) ||
        (rc = api_check_aligned(c.data, elem_size(out_type), "C")))
        return rc;
    return GK_OK;
}

// The written vector or matrix `w` meets none of what the call reads or writes besides.
int check_apart(const Span& w, const char* name, std::initializer_list<Span> others) {
    for (const Span& o : others)
        if (meet(w, o)) return api_err(GK_EINVAL, "gemmkit: %s aliases another operand", name);
    return GK_OK;
}

// Whether a 16-bit matrix can move in pairs: unit column stride, even rows of whole words.
bool in_pairs(const void* data, int64_t rs, int64_t cs, size_t rows, size_t cols) {
    return cols % 2 == 0 && cs == 1 && (rows <= 1 || (rs % 2 == 0 && rs < (int64_t{1} << 30))) &&
           (reinterpret_cast<uintptr_t>(data) & 3) == 0;
}

GroupedParams product_params(int is_f16, size_t groups, const int32_t* offsets, float alpha,
                             const gk_matref& a, const gk_matref& b, ptrdiff_t b_gs, const gk_matmut& c,
                             int out_type) {
    GroupedParams p;
    memset(&p, 0, sizeof(p));
    p.P = GOperand{static_cast<const uint16_t*>(b.data), b.cs, b.rs, groups > 1 ? b_gs : 0};
    p.Q = GOperand{static_cast<const uint16_t*>(a.data), a.rs, a.cs, 0};
    p.np = static_cast<int64_t>(b.cols);
    p.kdim = static_cast<int32_t>(a.cols);
    p.zero = a.cols == 0 || alpha == 0.0f;
    p.groups = static_cast<int>(groups);
    p.rows = static_cast<int>(a.rows);
    p.offsets = offsets;
    p.c = c.data;
    p.ldq = c.rs;
    p.ldp = c.cs;
    p.alpha = alpha;
    p.f16 = is_f16 != 0;
    p.out_type = out_type;
    return p;
}

// The backward entries' descriptor into p's epilogue; `in` are the matrices that the call reads.
int take_bwd(const gk_epilogue_bwd* d, int is_f16, size_t groups, const gk_matmut& c, int out_type,
             std::initializer_list<Span> in, EpiArgs* e) {
    int rc = check_act(d->act);
    if (rc) return rc;
    Span zs{nullptr, 0}, xs{nullptr, 0};
    e->act = d->act;
    e->slope = d->slope;
    const Span cs = span_of(c, elem_size(out_type));
    if (d->z8) {
        const gk_act8_matrix& q = *d->z8;
        if ((rc = check_act8(&q, "z"))) return rc;
        if (q.rows != c.rows || q.cols != c.cols)
            return api_err(GK_EINVAL, "gemmkit: z is %zux%zu, the output is %zux%zu", q.rows, q.cols,
                           c.rows, c.cols);
        zs = {q.codes, q.codes_len};
        xs = {q.exps, q.exps_len};
        e->z8 = Act8View{q.codes, q.exps, static_cast<int64_t>(q.codes_ld),
                         static_cast<int64_t>(q.exps_ld)};
        if (meet(cs, zs) || meet(cs, xs)) return api_err(GK_EINVAL, "gemmkit: C aliases z");
    } else if (d->z.data) {
        if ((rc = check_like_c(d->z, c, 2, "z"))) return rc;
        zs = span_of(d->z, 2);
        if (meet(cs, zs) && !(out_type != GK_F32 && same_view(d->z, c)))
            return api_err(GK_EINVAL, "gemmkit: C aliases z");
        e->side = d->z.data;
        e->sq = d->z.rs;
        e->sp = d->z.cs;
    } else if (d->act != GK_ACT_NONE) {
        return api_err(GK_EINVAL, "gemmkit: null z");
    }
    if (d->act == GK_ACT_NONE) {  // act' is 1: z is not read
        e->side = nullptr;
        e->z8 = Act8View{nullptr, nullptr, 0, 0};
    }
    if (d->dbias) {
        if ((rc = check_vector(d->dbias, d->dbias_len, d->dbias_gs, d->dbias_type, groups, c.cols, is_f16,
                               true, "dbias")))
            return rc;
        const Span ds{d->dbias, ((groups - 1) * d->dbias_gs + c.cols) * elem_size(d->dbias_type)};
        if ((rc = check_apart(ds, "dbias", {cs, zs, xs})) || (rc = check_apart(ds, "dbias", in)))
            return rc;
        e->dbias = d->dbias;
        e->dbias_gs = groups > 1 ? d->dbias_gs : 0;
        e->bias_type = d->dbias_type;
    }
    return GK_OK;
}

}  // namespace

}  // namespace gk

using namespace gk;

extern "C" {

int gk_gemm_half_epilogue(int is_f16, size_t groups, const int32_t* offsets, float alpha,
                          gk_matref a, gk_matref b, ptrdiff_t b_gs, const gk_epilogue* epi,
                          gk_matmut c, int out_type, gk_parallelism par, gk_stream_t stream) {
    (void)par;
    if (!epi) return api_err(GK_EINVAL, "gemmkit: null epilogue");
    int rc = check_product(is_f16, groups, offsets, a, b, b_gs, c, out_type);
    if (rc || (rc = check_act(epi->act))) return rc;
    const size_t so = elem_size(out_type);
    const Span cs = span_of(c, so), as{a.data, a.len * 2}, bs{b.data, b.len * 2};
    GroupedParams p = product_params(is_f16, groups, offsets, alpha, a, b, b_gs, c, out_type);
    EpiArgs& e = p.e;
    e.act = epi->act;
    e.slope = epi->slope;
    Span vs{nullptr, 0}, rs{nullptr, 0};
    if (epi->bias) {
        if ((rc = check_vector(epi->bias, epi->bias_len, epi->bias_gs, epi->bias_type, groups, c.cols,
                               is_f16, false, "bias")))
            return rc;
        e.bias = epi->bias;
        e.bias_gs = groups > 1 ? epi->bias_gs : 0;
        e.bias_type = epi->bias_type;
        vs = {epi->bias, ((groups - 1) * epi->bias_gs + c.cols) * elem_size(epi->bias_type)};
        if ((rc = check_apart(cs, "C", {vs}))) return rc;
    }
    if (epi->residual.data) {
        if ((rc = check_like_c(epi->residual, c, so, "the residual"))) return rc;
        rs = span_of(epi->residual, so);
        if (meet(cs, rs) && !same_view(epi->residual, c))
            return api_err(GK_EINVAL, "gemmkit: C aliases the residual");
        e.side = epi->residual.data;
        e.sq = epi->residual.rs;
        e.sp = epi->residual.cs;
    }
    if (epi->z.data) {
        const gk_matref z{epi->z.data, epi->z.len, epi->z.rows, epi->z.cols, epi->z.rs, epi->z.cs};
        if ((rc = check_like_c(z, c, 2, "z"))) return rc;
        if (api_self_aliases(z.rows, z.cols, z.rs, z.cs))
            return api_err(GK_EINVAL, "gemmkit: z view aliases itself");
        if ((rc = check_apart(span_of(z, 2), "z", {cs, as, bs, vs, rs}))) return rc;
        e.z = static_cast<uint16_t*>(epi->z.data);
        e.zq = z.rs;
        e.zp = z.cs;
    }
    if (c.rows == 0 || c.cols == 0) return GK_OK;
    if (!c.data) return api_err(GK_EINVAL, "gemmkit: null C");
    if (!p.zero && (!a.data || !b.data)) return api_err(GK_EINVAL, "gemmkit: null A or B");
    e.pairs = out_type != GK_F32 && in_pairs(c.data, c.rs, c.cs, c.rows, c.cols) &&
              (!e.side || in_pairs(e.side, e.sq, e.sp, c.rows, c.cols)) &&
              (!e.z || in_pairs(e.z, e.zq, e.zp, c.rows, c.cols));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return p.f16 ? run_grouped<EPI_FWD | EPI_F16>(p, st) : run_grouped<EPI_FWD>(p, st);
}

int gk_gemm_half_dact(int is_f16, size_t groups, const int32_t* offsets, float alpha, gk_matref a,
                      gk_matref b, ptrdiff_t b_gs, const gk_epilogue_bwd* epi, gk_matmut c,
                      int out_type, gk_parallelism par, gk_stream_t stream) {
    (void)par;
    if (!epi) return api_err(GK_EINVAL, "gemmkit: null epilogue");
    int rc = check_product(is_f16, groups, offsets, a, b, b_gs, c, out_type);
    if (rc) return rc;
    GroupedParams p = product_params(is_f16, groups, offsets, alpha, a, b, b_gs, c, out_type);
    const Span as{a.data, a.len * 2}, bs{b.data, b.len * 2};
    if ((rc = take_bwd(epi, is_f16, groups, c, out_type, {as, bs}, &p.e))) return rc;
    if (c.cols == 0) return GK_OK;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c.rows == 0) {
        if (!p.e.dbias) return GK_OK;
        int dev = 0;
        if ((rc = api_check_device(&dev))) return rc;
        return launch_sum_parts(nullptr, nullptr, p.groups, 0, 1, 1, 0, p.np, p.e, st);
    }
    if (!c.data) return api_err(GK_EINVAL, "gemmkit: null C");
    if (!p.zero && (!a.data || !b.data)) return api_err(GK_EINVAL, "gemmkit: null A or B");
    p.e.pairs = out_type != GK_F32 && in_pairs(c.data, c.rs, c.cs, c.rows, c.cols) &&
                (!p.e.side || in_pairs(p.e.side, p.e.sq, p.e.sp, c.rows, c.cols));
    return p.f16 ? run_grouped<EPI_BWD | EPI_F16>(p, st) : run_grouped<EPI_BWD>(p, st);
}

int gk_act_backward(int is_f16, size_t groups, const int32_t* offsets, gk_matref dy,
                    const gk_epilogue_bwd* epi, gk_matmut dz, int out_type, gk_stream_t stream) {
    if (!epi) return api_err(GK_EINVAL, "gemmkit: null epilogue");
    static const int32_t all = 0;
    if (!offsets && groups != 1) return api_err(GK_EINVAL, "gemmkit: null offsets");
    int rc = check_groups(groups, offsets ? offsets : &all, dy.rows, is_f16, out_type);
    if (rc) return rc;
    if ((rc = api_check_view(dy.len, dy.rows, dy.cols, dy.rs, dy.cs, "dY")) ||
        (rc = api_check_aligned(dy.data, 2, "dY")))
        return rc;
    if (dy.cols > INT32_MAX / 2)
        return api_err(GK_EINVAL, "gemmkit: problem dimensions exceed the engine's limits");
    const size_t so = elem_size(out_type);
    const Span ys = span_of(dy, 2);
    if (dz.data) {
        if (dz.rows != dy.rows || dz.cols != dy.cols)
            return api_err(GK_EINVAL, "gemmkit: dZ is %zux%zu, dY is %zux%zu", dz.rows, dz.cols, dy.rows,
                           dy.cols);
        if ((rc = api_check_view(dz.len, dz.rows, dz.cols, dz.rs, dz.cs, "dZ")) ||
            (rc = api_check_aligned(dz.data, so, "dZ")))
            return rc;
        if (api_self_aliases(dz.rows, dz.cols, dz.rs, dz.cs))
            return api_err(GK_EINVAL, "gemmkit: dZ view aliases itself");
        if (meet(span_of(dz, so), ys) && !(out_type != GK_F32 && same_view(dy, dz)))
            return api_err(GK_EINVAL, "gemmkit: dZ aliases dY");
    } else {
        if (!epi->dbias) return api_err(GK_EINVAL, "gemmkit: neither dZ nor dbias");
        dz = gk_matmut{nullptr, 0, dy.rows, dy.cols, 0, 0};
    }
    ActGrad p;
    memset(&p, 0, sizeof(p));
    if ((rc = take_bwd(epi, is_f16, groups, dz, out_type, {ys}, &p.e))) return rc;
    if (dy.cols == 0) return GK_OK;
    if (dy.rows && !dy.data) return api_err(GK_EINVAL, "gemmkit: null dY");
    if (!p.e.dbias && dy.rows == 0) return GK_OK;
    int dev = 0;
    if ((rc = api_check_device(&dev))) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int rows = static_cast<int>(dy.rows);
    p.dy = static_cast<const uint16_t*>(dy.data);
    p.yq = dy.rs;
    p.yp = dy.cs;
    p.dz = dz.data;
    p.zq = dz.rs;
    p.zp = dz.cs;
    p.np = static_cast<int64_t>(dy.cols);
    p.offsets = offsets;
    p.groups = static_cast<int>(groups);
    p.rows = rows;
    p.f16 = is_f16 != 0;
    p.out_type = out_type;
    p.status = device_status_ptr();
    void* scratch = nullptr;
    if (rows) {
        auto whole = [&](const void* d, int64_t rs, int64_t cs, size_t es) {
            return cs == 1 && (rows == 1 || rs * es % 16 == 0) &&
                   (reinterpret_cast<uintptr_t>(d) & 15) == 0;
        };
        const bool vec = p.np % 8 == 0 && whole(p.dy, p.yq, p.yp, 2) &&
                         (!p.dz || whole(p.dz, p.zq, p.zp, so)) &&
                         (!p.e.side || whole(p.e.side, p.e.sq, p.e.sp, 2));
        const int64_t wide = vec ? 256 : 32, blocks = (p.np + wide - 1) / wide;
        // slices: what makes the grid resident at once, of 32 rows at least
        int64_t slices = 3ll * sm_count() / blocks;
        if (slices < 1) slices = 1;
        int64_t slice = (rows + slices - 1) / slices;
        slice = slice < 32 ? 32 : slice;
        slices = (rows + slice - 1) / slice;
        p.slice = static_cast<int>(slice);
        if (p.e.dbias && (rc = scratch_alloc(&scratch, static_cast<size_t>(slices + p.groups) * p.np * 4, st)))
            return rc;
        p.part = static_cast<float*>(scratch);
        rc = launch_overlapped(p.f16 ? act_grad_for<true>(vec, p.e.act) : act_grad_for<false>(vec, p.e.act),
                               dim3(static_cast<unsigned>(slices * blocks)), 32 * GW, st, p);
    }
    if (!rc && p.e.dbias)
        rc = launch_sum_parts(p.part, offsets, p.groups, rows, 1, 1, p.slice, p.np, p.e, st);
    const int fr = scratch_free(scratch, st);
    return rc ? rc : fr;
}

}  // extern "C"
