// The residual step between the blocks of a context network, with the norms behind one block and before the next:
//   z = norm(f; post)  (or f),   y = x + scale * gate * z,   u = norm(y; pre)  (or none),
//   norm = (v - mean) rsqrt(var + eps) w + b  (layer)  or  v rsqrt(mean(v^2) + eps) w  + b (rms).
// One pass over memory: a row stays in the registers of L threads (8, 64, 256, 512 or 1024) from its loads to its stores, so the forward
// moves x, f, y, u once and the backward x, f, grad_y, grad_u, grad_x, grad_f once -- the backward recomputes both norms from x and f
// instead of reading anything the forward kept.  Bound: HBM.  All sums are fp32, the spread is taken about the mean (two sums), y
// enters the second norm before its rounding to the output type.
// Parameter gradients are column sums: every workgroup sums its rows in registers, norm_columns_kernel adds the workgroups' partial
// rows in order.  The gate's gradient is a sum over the rows that share a gate row: a workgroup takes whole runs of them.
#include "planes.h"

namespace eq {

constexpr int kNormMaxWidth = 8192;

struct NormShape {
    int64_t rows;
    int width;
    int64_t gate_rows;                        // rows that share one row of the gate (rows when there is one gate row; unused without a gate)
    int rms, post, pre;
    float eps;
    float factor;                             // a constant residual scale
    const float *post_w, *post_b, *pre_w, *pre_b, *scale;      // [width] each, may be null
};

template <int T>
struct NormArgs {
    using E = typename Num<T>::type;
    NormShape s;
    const E *x, *f, *gate;
    E *y, *u;
    const E *gy, *gu;                         // either may be null
    E *gx, *gf;                               // either may be null
    E* ggate;                                 // [rows / gate_rows, width] or null
    float* part;                              // [5][blocks][width]: pre_w, pre_b, post_w, post_b, scale
    float* gate_part;                         // [units][width] when a gate row's rows are cut
    int64_t units;                            // (gate row, run of rows) pairs, or runs of rows
    int unit_rows, cuts;                      // rows of a unit; units of one gate row
    int want;                                 // bit i: partial i is wanted; bit 5: the gate's gradient
};

// L threads own a row, PER chunks of eight columns each; NT threads of a workgroup own NT / L rows at a time
template <int L, int NT>
__device__ __forceinline__ float row_sum(float v, float* lds) {
    if constexpr (L <= 64) {
#pragma unroll
        for (int o = L / 2; o; o >>= 1) v += __shfl_xor(v, o);
        return v;
    } else {
#pragma unroll
        for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
        __syncthreads();                      // the previous sum has been read
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) t += lds[i];
        return t;
    }
}

template <int T, int L, int PER>
struct Row {
    float v[PER * 8];
    __device__ __forceinline__ void load(const typename Num<T>::type* row, int width, int t) {
#pragma unroll
        for (int c = 0; c < PER; ++c) {
            const int col = (c * L + t) * 8;
            const Raw8<T> r = row && col < width ? load8<T>(row, col, width) : raw_zero<T>();
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c * 8 + i] = raw_float<T>(r, i);
        }
    }
    __device__ __forceinline__ void store(typename Num<T>::type* row, int width, int t) const {
#pragma unroll
        for (int c = 0; c < PER; ++c) {
            const int col = (c * L + t) * 8;
            if (col < width) {
                float a[4], b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) { a[i] = v[c * 8 + i]; b[i] = v[c * 8 + 4 + i]; }
                store4<T>(row + col, a, width - col);
                if (col + 4 < width) store4<T>(row + col + 4, b, width - col - 4);
            }
        }
    }
};

template <int L, int PER>
__device__ __forceinline__ void load_columns(float (&w)[PER * 8], const float* p, int width, int t, float otherwise) {
#pragma unroll
    for (int c = 0; c < PER; ++c) {
        const int col = (c * L + t) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[c * 8 + i] = otherwise;
        if (p && col < width) {
            const Raw8<kF32> r = load8<kF32>(p, col, width);
#pragma unroll
            for (int i = 0; i < 8; ++i) w[c * 8 + i] = raw_float<kF32>(r, i);
        }
    }
}

// v -> its unit row in place (columns behind the width become zero); returns 1 / spread
template <int L, int PER, int NT>
__device__ __forceinline__ float unit_row(float (&v)[PER * 8], int rms, float eps, int width, int t, float* lds) {
    const float inv = 1.f / (float)width;
    if (!rms) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < PER * 8; ++i) sum += v[i];
        const float mean = row_sum<L, NT>(sum, lds) * inv;
#pragma unroll
        for (int c = 0; c < PER; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c * 8 + i] = (c * L + t) * 8 + i < width ? v[c * 8 + i] - mean : 0.f;
    }
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < PER * 8; ++i) sq = fmaf(v[i], v[i], sq);
    const float r = 1.f / sqrtf(row_sum<L, NT>(sq, lds) * inv + eps);
#pragma unroll
    for (int i = 0; i < PER * 8; ++i) v[i] *= r;
    return r;
}

template <int T, int L, int PER, int NT>
__global__ __launch_bounds__(NT) void norm_fwd_kernel(NormArgs<T> a) {
    const NormShape& s = a.s;
    __shared__ float lds[NT / 64];
    const int t = threadIdx.x % L;
    const int64_t step = (int64_t)gridDim.x * (NT / L);
    for (int64_t r0 = (int64_t)blockIdx.x * (NT / L); r0 < s.rows; r0 += step) {
        const int64_t row = r0 + threadIdx.x / L;
        const bool ok = row < s.rows;
        const int64_t at = row * s.width;
        Row<T, L, PER> x, f;
        x.load(ok ? a.x + at : nullptr, s.width, t);
        f.load(ok && a.f ? a.f + at : nullptr, s.width, t);
        float w[PER * 8];
        if (s.post) {
            unit_row<L, PER, NT>(f.v, s.rms, s.eps, s.width, t, lds);
            load_columns<L, PER>(w, s.post_w, s.width, t, 1.f);
#pragma unroll
            for (int i = 0; i < PER * 8; ++i) f.v[i] *= w[i];
            if (s.post_b) {
                load_columns<L, PER>(w, s.post_b, s.width, t, 0.f);
#pragma unroll
                for (int i = 0; i < PER * 8; ++i) f.v[i] += w[i];
            }
        }
        load_columns<L, PER>(w, s.scale, s.width, t, s.factor);
        if (a.gate) {
            Row<T, L, PER> g;
            g.load(ok ? a.gate + row / s.gate_rows * s.width : nullptr, s.width, t);
#pragma unroll
            for (int i = 0; i < PER * 8; ++i) w[i] *= g.v[i];
        }
#pragma unroll
        for (int i = 0; i < PER * 8; ++i) x.v[i] = fmaf(w[i], f.v[i], x.v[i]);
        if (ok && a.y) x.store(a.y + at, s.width, t);
        if (s.pre) {
            unit_row<L, PER, NT>(x.v, s.rms, s.eps, s.width, t, lds);
            load_columns<L, PER>(w, s.pre_w, s.width, t, 1.f);
#pragma unroll
            for (int i = 0; i < PER * 8; ++i) x.v[i] *= w[i];
            if (s.pre_b) {
                load_columns<L, PER>(w, s.pre_b, s.width, t, 0.f);
#pragma unroll
                for (int i = 0; i < PER * 8; ++i) x.v[i] += w[i];
            }
            if (ok) x.store(a.u + at, s.width, t);
        }
    }
}

// g <- gradient of the rows whose unit rows are n: (g - [layer: mean g] - n mean(g n)) r
template <int L, int PER, int NT>
__device__ __forceinline__ void unit_row_grad(float (&g)[PER * 8], const float (&n)[PER * 8], float r, int rms, int width, int t, float* lds) {
    const float inv = 1.f / (float)width;
    float sg = 0.f, sn = 0.f;
#pragma unroll
    for (int i = 0; i < PER * 8; ++i) { sg += g[i]; sn = fmaf(g[i], n[i], sn); }
    sn = row_sum<L, NT>(sn, lds) * inv;
    sg = rms ? 0.f : row_sum<L, NT>(sg, lds) * inv;
#pragma unroll
    for (int c = 0; c < PER; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = c * 8 + i;
            g[k] = (c * L + t) * 8 + i < width ? (g[k] - sg - n[k] * sn) * r : 0.f;
        }
}

// sums acc over the row groups of the workgroup and writes (or rounds) one row of width values
template <int L, int PER, int NT, class F>
__device__ __forceinline__ void group_columns(const float (&acc)[PER * 8], float* lds, int width, F put) {
    const int t = threadIdx.x % L, grp = threadIdx.x / L;
    if constexpr (NT == L) {
#pragma unroll
        for (int c = 0; c < PER; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((c * L + t) * 8 + i < width) put((c * L + t) * 8 + i, acc[c * 8 + i]);
    } else {
        constexpr int kCols = L * PER * 8;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < PER; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) lds[grp * kCols + (c * L + t) * 8 + i] = acc[c * 8 + i];
        __syncthreads();
        for (int col = threadIdx.x; col < width; col += NT) {
            float v = 0.f;
            for (int q = 0; q < NT / L; ++q) v += lds[q * kCols + col];
            put(col, v);
        }
    }
}

template <int T, int L, int PER, int NT>
__global__ __launch_bounds__(NT) void norm_bwd_kernel(NormArgs<T> a) {
    constexpr int V = PER * 8, G = NT / L;
    const NormShape& s = a.s;
    __shared__ float lds[NT / 64];
    __shared__ float cols[G > 1 ? G * L * V : 1];
    const int t = threadIdx.x % L;
    float s_prew[V], s_preb[V], s_postw[V], s_postb[V], s_scale[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s_prew[i] = s_preb[i] = s_postw[i] = s_postb[i] = s_scale[i] = 0.f;
    for (int64_t unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        const int64_t gate_row = unit / a.cuts, first = gate_row * s.gate_rows + (unit - gate_row * a.cuts) * a.unit_rows;
        const int64_t group_end = (gate_row + 1) * s.gate_rows, end0 = first + a.unit_rows, end = end0 < group_end ? end0 : group_end;
        float s_gate[V];
#pragma unroll
        for (int i = 0; i < V; ++i) s_gate[i] = 0.f;
        for (int64_t r0 = first; r0 < end; r0 += G) {
            const int64_t row = r0 + threadIdx.x / L, at = row * s.width;
            const bool ok = row < end && row < s.rows;
            Row<T, L, PER> x, f, gu, gy;
            f.load(ok && a.f ? a.f + at : nullptr, s.width, t);
            x.load(ok ? a.x + at : nullptr, s.width, t);
            gu.load(ok && a.gu ? a.gu + at : nullptr, s.width, t);
            gy.load(ok && a.gy ? a.gy + at : nullptr, s.width, t);
            float w[V], z[V], fr = 1.f;
            if (s.post) {
                fr = unit_row<L, PER, NT>(f.v, s.rms, s.eps, s.width, t, lds);
                load_columns<L, PER>(w, s.post_w, s.width, t, 1.f);
#pragma unroll
                for (int i = 0; i < V; ++i) z[i] = f.v[i] * w[i];
                if (s.post_b) {
                    load_columns<L, PER>(w, s.post_b, s.width, t, 0.f);
#pragma unroll
                    for (int i = 0; i < V; ++i) z[i] += w[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) z[i] = f.v[i];
            }
            float sc[V];
            Row<T, L, PER> gt;
            load_columns<L, PER>(sc, s.scale, s.width, t, s.factor);
            if (a.gate) gt.load(ok ? a.gate + gate_row * s.width : nullptr, s.width, t);
            else
#pragma unroll
                for (int i = 0; i < V; ++i) gt.v[i] = 1.f;
            if (s.pre) {
#pragma unroll
                for (int i = 0; i < V; ++i) x.v[i] = fmaf(sc[i] * gt.v[i], z[i], x.v[i]);
                const float yr = unit_row<L, PER, NT>(x.v, s.rms, s.eps, s.width, t, lds);
                load_columns<L, PER>(w, s.pre_w, s.width, t, 1.f);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s_prew[i] = fmaf(gu.v[i], x.v[i], s_prew[i]);
                    s_preb[i] += gu.v[i];
                    gu.v[i] *= w[i];
                }
                unit_row_grad<L, PER, NT>(gu.v, x.v, yr, s.rms, s.width, t, lds);
#pragma unroll
                for (int i = 0; i < V; ++i) gy.v[i] += gu.v[i];
            }
            if (ok && a.gx) gy.store(a.gx + at, s.width, t);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float gz = gy.v[i] * z[i];
                s_gate[i] = fmaf(gz, sc[i], s_gate[i]);
                s_scale[i] = fmaf(gz, gt.v[i], s_scale[i]);
                gy.v[i] *= sc[i] * gt.v[i];
            }
            if (s.post) {
                load_columns<L, PER>(w, s.post_w, s.width, t, 1.f);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s_postw[i] = fmaf(gy.v[i], f.v[i], s_postw[i]);
                    s_postb[i] += gy.v[i];
                    gy.v[i] *= w[i];
                }
                if (a.gf) unit_row_grad<L, PER, NT>(gy.v, f.v, fr, s.rms, s.width, t, lds);
            }
            if (ok && a.gf) gy.store(a.gf + at, s.width, t);
        }
        if (a.want & 32) {
            if (a.cuts == 1) group_columns<L, PER, NT>(s_gate, cols, s.width, [&](int c, float v) { store_value<T>(a.ggate + gate_row * s.width + c, v); });
            else group_columns<L, PER, NT>(s_gate, cols, s.width, [&](int c, float v) { a.gate_part[unit * s.width + c] = v; });
        }
    }
    auto put = [&](int k, const float (&acc)[V]) {
        if (a.want >> k & 1)
            group_columns<L, PER, NT>(acc, cols, s.width, [&](int c, float v) { a.part[((int64_t)k * gridDim.x + blockIdx.x) * s.width + c] = v; });
    };
    put(0, s_prew);
    put(1, s_preb);
    put(2, s_postw);
    put(3, s_postb);
    put(4, s_scale);
}

struct NormColumns { float* out[5]; };

// out[k] = sum over the workgroups' partial rows, in order: 64 columns x 4 runs of rows per workgroup
__global__ __launch_bounds__(256) void norm_columns_kernel(const float* part, int parts, int width, NormColumns o) {
    __shared__ float lds[4][64];
    const int k = blockIdx.y, c = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
    if (!o.out[k]) return;
    float v = 0.f;
    if (c < width)
        for (int p = q; p < parts; p += 4) v += part[((int64_t)k * parts + p) * width + c];
    lds[q][threadIdx.x & 63] = v;
    __syncthreads();
    if (q == 0 && c < width) o.out[k][c] = (lds[0][threadIdx.x] + lds[1][threadIdx.x]) + (lds[2][threadIdx.x] + lds[3][threadIdx.x]);
}

// a gate row's gradient from its cuts, in order
template <int T>
__global__ __launch_bounds__(256) void norm_gate_kernel(const float* part, int cuts, int width, typename Num<T>::type* out) {
    const int64_t g = blockIdx.y;
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= width) return;
    float v = 0.f;
    for (int p = 0; p < cuts; ++p) v += part[(g * cuts + p) * width + c];
    store_value<T>(out + g * width + c, v);
}

// threads of a row and of a workgroup by the width: the row fits the registers, narrow rows share a wave
static int norm_group_rows(int width) { return width <= 64 ? 32 : width <= 512 ? 4 : 1; }

struct NormPlan { int64_t units; int unit_rows, cuts, blocks; };
// Backward: up to 1024 workgroups.  With a gate, a unit is a run of rows of one gate row (a gate row with many rows is cut); without,
// a run of rows.
static NormPlan norm_plan(const NormShape& s, bool gated) {
    NormPlan p;
    const int g = norm_group_rows(s.width);
    const int64_t groups = s.rows / s.gate_rows, most = 1024;
    int64_t cuts = groups >= most ? 1 : most / groups;
    const int64_t room = (s.gate_rows + g - 1) / g;
    if (cuts > room) cuts = room;
    p.unit_rows = (int)((room + cuts - 1) / cuts * g);
    p.cuts = (int)((s.gate_rows + p.unit_rows - 1) / p.unit_rows);
    p.units = groups * p.cuts;
    p.blocks = (int)(p.units < most ? p.units : most);
    return p;
}

template <int T>
static int norm_run(const NormArgs<T>& a, bool backward, int blocks, hipStream_t st) {
    const int w = a.s.width;
#define EQ_NORM(L, PER, NT)                                                            \
    do {                                                                               \
        if (backward) norm_bwd_kernel<T, L, PER, NT><<<blocks, NT, 0, st>>>(a);        \
        else norm_fwd_kernel<T, L, PER, NT><<<blocks, NT, 0, st>>>(a);                 \
    } while (0)
    if (w <= 64) EQ_NORM(8, 1, 256);
    else if (w <= 512) EQ_NORM(64, 1, 256);
    else if (w <= 2048) EQ_NORM(256, 1, 256);
    else if (w <= 4096) EQ_NORM(512, 1, 512);
    else EQ_NORM(1024, 1, 1024);
#undef EQ_NORM
    EQ_CHECK_LAUNCH(backward ? "residual_norm_backward" : "residual_norm_forward");
    return 0;
}

static int norm_shape(const equigspr_residual_norm* d, NormShape* s) {
    EQ_CHECK_ARG(d, EQUIGSPR_EINVAL, "residual_norm: null description");
    EQ_CHECK_ARG(d->dtype == EQUIGSPR_F32 || d->dtype == EQUIGSPR_BF16 || d->dtype == EQUIGSPR_F16, EQUIGSPR_EINVAL, "residual_norm: unknown dtype %d", d->dtype);
    EQ_CHECK_ARG(d->rows >= 0 && d->rows < (1ll << 40), EQUIGSPR_EINVAL, "residual_norm: bad number of rows");
    EQ_CHECK_ARG(d->width >= 1 && d->width <= kNormMaxWidth, EQUIGSPR_ENOTSUP, "residual_norm: width %d, the kernels take 1..%d", d->width, kNormMaxWidth);
    EQ_CHECK_ARG(d->eps >= 0.f && d->eps < INFINITY, EQUIGSPR_EINVAL, "residual_norm: eps must be finite and not negative");
    EQ_CHECK_ARG(!d->gate || (d->gate_rows >= 1 && d->rows % d->gate_rows == 0), EQUIGSPR_EINVAL, "residual_norm: the gate's rows do not divide the rows");
    EQ_CHECK_ARG(d->rows == 0 || d->x, EQUIGSPR_EINVAL, "residual_norm: null tensor");
    EQ_CHECK_ARG(d->f || (d->pre_weight && !d->gate && !d->scale && !d->post_weight), EQUIGSPR_EINVAL,
                 "residual_norm: without f there is only the norm before the next block");
    s->rows = d->rows; s->width = d->width; s->rms = d->rms != 0; s->eps = d->eps; s->factor = d->factor;
    s->gate_rows = d->gate ? d->gate_rows : (d->rows ? d->rows : 1);
    s->post = d->post_weight != nullptr; s->pre = d->pre_weight != nullptr;
    s->post_w = d->post_weight; s->post_b = s->post ? d->post_bias : nullptr;
    s->pre_w = d->pre_weight; s->pre_b = s->pre ? d->pre_bias : nullptr;
    s->scale = d->scale;
    return 0;
}

template <int T>
static int norm_forward(const equigspr_residual_norm* d, const NormShape& s, void* y, void* u, hipStream_t st) {
    using E = typename Num<T>::type;
    NormArgs<T> a = {};
    a.s = s;
    a.x = (const E*)d->x; a.f = (const E*)d->f; a.gate = (const E*)d->gate;
    a.y = (E*)y; a.u = (E*)u;
    const int64_t groups = (s.rows + norm_group_rows(s.width) - 1) / norm_group_rows(s.width);
    return norm_run<T>(a, false, (int)(groups < 8192 ? groups : 8192), st);
}

template <int T>
static int norm_backward(const equigspr_residual_norm* d, const NormShape& s, const void* gy, const void* gu, float* work, const equigspr_residual_norm_grads* o,
                         hipStream_t st) {
    using E = typename Num<T>::type;
    NormArgs<T> a = {};
    a.s = s;
    a.x = (const E*)d->x; a.f = (const E*)d->f; a.gate = (const E*)d->gate;
    a.gy = (const E*)gy; a.gu = (const E*)gu;
    a.gx = (E*)o->grad_x; a.gf = (E*)o->grad_f; a.ggate = a.gate ? (E*)o->grad_gate : nullptr;
    const NormPlan p = norm_plan(s, a.gate != nullptr);
    a.units = p.units; a.unit_rows = p.unit_rows; a.cuts = p.cuts;
    NormColumns c = {{s.pre ? o->grad_pre_weight : nullptr, s.pre ? o->grad_pre_bias : nullptr, s.post ? o->grad_post_weight : nullptr,
                      s.post ? o->grad_post_bias : nullptr, o->grad_scale}};
    for (int k = 0; k < 5; ++k) a.want |= c.out[k] ? 1 << k : 0;
    const bool columns = a.want != 0;
    if (a.ggate) a.want |= 32;
    a.part = work;
    a.gate_part = work + (int64_t)5 * p.blocks * s.width;
    if (const int rc = norm_run<T>(a, true, p.blocks, st)) return rc;
    if (columns) {
        norm_columns_kernel<<<dim3(ceil_div(s.width, 64), 5), 256, 0, st>>>(a.part, p.blocks, s.width, c);
        EQ_CHECK_LAUNCH("residual_norm_backward (columns)");
    }
    if (a.ggate && p.cuts > 1) {
        norm_gate_kernel<T><<<dim3(ceil_div(s.width, 256), (unsigned)(s.rows / s.gate_rows)), 256, 0, st>>>(a.gate_part, p.cuts, s.width, a.ggate);
        EQ_CHECK_LAUNCH("residual_norm_backward (gate)");
    }
    return 0;
}

}  // namespace eq

extern "C" int equigspr_residual_norm_forward(const equigspr_residual_norm* d, void* y, void* u, void* stream) {
    eq::NormShape s;
    if (const int rc = eq::norm_shape(d, &s)) return rc;
    if (s.rows == 0) return 0;
    EQ_CHECK_ARG((y || !d->f) && (u || !s.pre), EQUIGSPR_EINVAL, "residual_norm_forward: null output");
    hipStream_t st = (hipStream_t)stream;
    switch (d->dtype) {
        case EQUIGSPR_F32: return eq::norm_forward<eq::kF32>(d, s, y, u, st);
        case EQUIGSPR_BF16: return eq::norm_forward<eq::kBF16>(d, s, y, u, st);
        default: return eq::norm_forward<eq::kF16>(d, s, y, u, st);
    }
}

extern "C" int64_t equigspr_residual_norm_backward_work_size(const equigspr_residual_norm* d) {
    eq::NormShape s;
    if (eq::norm_shape(d, &s) != 0) return -1;
    if (s.rows == 0) return 0;
    const eq::NormPlan p = eq::norm_plan(s, d->gate != nullptr);
    return ((int64_t)5 * p.blocks + (d->gate && p.cuts > 1 ? p.units : 0)) * s.width;
}

extern "C" int equigspr_residual_norm_backward(const equigspr_residual_norm* d, const void* grad_y, const void* grad_u, float* work,
                                               const equigspr_residual_norm_grads* out, void* stream) {
    eq::NormShape s;
    if (const int rc = eq::norm_shape(d, &s)) return rc;
    if (s.rows == 0) return 0;
    EQ_CHECK_ARG(out && work, EQUIGSPR_EINVAL, "residual_norm_backward: null gradients or work");
    hipStream_t st = (hipStream_t)stream;
    switch (d->dtype) {
        case EQUIGSPR_F32: return eq::norm_backward<eq::kF32>(d, s, grad_y, grad_u, work, out, st);
        case EQUIGSPR_BF16: return eq::norm_backward<eq::kBF16>(d, s, grad_y, grad_u, work, out, st);
        default: return eq::norm_backward<eq::kF16>(d, s, grad_y, grad_u, work, out, st);
    }
}
