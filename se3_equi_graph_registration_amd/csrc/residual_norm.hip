// The residual step between the blocks of a context network, with the norms behind one block and before the next:
//   z = norm(f; post)  (or f),   y = x + scale * gate * z,   u = norm(y; pre)  (or none),
//   norm = (v - mean) rsqrt(var + eps) w + b  (layer)  or  v rsqrt(mean(v^2) + eps) w  + b (rms).
// One pass over memory: a row stays in the registers of L threads (8, 64, 256, 512 or 1024) from its loads to its stores, so the forward
// moves x, f, y, u once and the backward x, f, grad_y, grad_u, grad_x, grad_f once -- the backward recomputes both norms from x and f
// instead of reading anything the forward kept.  (The backward of widths above 4096 has 128 registers a thread and spills 77..147 of them:
// 224..288 bytes of scratch; a few are spilled where odd widths cut the columns.)  Bound: HBM forward
// (32768 x 2048 bf16: 111 us, 4.8 TB/s); backward the registers of its column sums, which leave two workgroups per compute unit (250 us,
// 3.2 TB/s), and above 4096 the spills (8192 x 8192 bf16: training 744 us, 156 of them forward).  A gate of x's shape makes every row
// a unit with sums of its own: 131072 x 64 bf16, training, 650 us against 95 with a gate per sample, 32768 x 2048 448 against 293.
// All sums are fp32, the spread is taken about the mean (two sums), y enters the second norm before its rounding to the output type.
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

// L threads own a row, eight consecutive columns each; NT threads of a workgroup own NT / L rows at a time.  Sums over a row: one meeting
// of the workgroup each (two buffers in turn: whoever writes one again has met everybody since they read it).
template <int L, int NT>
struct RowSums {
    float* lds;                               // [2][2][NT / 64]
    int turn;
    __device__ __forceinline__ void sum(float& a, float& b) {
#pragma unroll
        for (int o = (L < 64 ? L : 64) / 2; o; o >>= 1) { a += __shfl_xor(a, o); b += __shfl_xor(b, o); }
        if constexpr (L > 64) {
            float* s = lds + turn * 2 * (NT / 64);
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) { s[threadIdx.x >> 6] = a; s[NT / 64 + (threadIdx.x >> 6)] = b; }
            __syncthreads();
            a = b = 0.f;
#pragma unroll
            for (int i = 0; i < NT / 64; ++i) { a += s[i]; b += s[NT / 64 + i]; }
        }
    }
    __device__ __forceinline__ float sum(float a) {
        float b = 0.f;
        sum(a, b);
        return a;
    }
};

// kEven: width % 8 == 0, no thread's columns are cut (the code for cut ones spills the kernels' scalar registers)
template <int T, bool kEven>
__device__ __forceinline__ Raw8<T> load_row(const typename Num<T>::type* row, int width, int col) {
    if constexpr (kEven) return row && col < width ? load8<T>(row + col, 0, 8) : raw_zero<T>();
    else return row && col < width ? load8_small<T>(row, col, width) : raw_zero<T>();
}
template <int T>
__device__ __forceinline__ void row_values(const Raw8<T>& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = raw_float<T>(r, i);
}
template <bool kEven>
__device__ __forceinline__ void load_columns(const float* p, int width, int col, float otherwise, float (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = otherwise;
    if (p && col < width) row_values<kF32>(load_row<kF32, kEven>(p, width, col), w);
}

// v -> its unit row in place (columns behind the width become zero); returns 1 / spread
template <bool kRms, class S>
__device__ __forceinline__ float unit_row(float (&v)[8], float eps, int width, int col, S& sums) {
    const float inv = 1.f / (float)width;
    if constexpr (!kRms) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += v[i];
        const float mean = sums.sum(sum) * inv;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < width ? v[i] - mean : 0.f;
    }
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sq = fmaf(v[i], v[i], sq);
    const float r = 1.f / sqrtf(sums.sum(sq) * inv + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= r;
    return r;
}

// g <- gradient of the rows whose unit rows are n: (g - [layer: mean g] - n mean(g n)) r
template <bool kRms, class S>
__device__ __forceinline__ void unit_row_grad(float (&g)[8], const float (&n)[8], float r, int width, int col, S& sums) {
    const float inv = 1.f / (float)width;
    float sg = 0.f, sn = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (!kRms) sg += g[i];
        sn = fmaf(g[i], n[i], sn);
    }
    sums.sum(sn, sg);
    sn *= inv;
    sg *= inv;
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = col + i < width ? (g[i] - (kRms ? 0.f : sg) - n[i] * sn) * r : 0.f;
}

// The parameters of a thread's columns stay in registers while it walks its rows, and the next row is loaded under this row's arithmetic;
// the widest rows (1024 threads, 128 registers each) have no room for either.
template <int T, int L, int NT, bool kRms, bool kEven>
__global__ __launch_bounds__(NT) void norm_fwd_kernel(NormArgs<T> a) {
    constexpr bool kAhead = NT < 1024;
    const NormShape& s = a.s;
    __shared__ float lds[4 * (NT / 64)];
    RowSums<L, NT> sums = {lds, 0};
    const int col = threadIdx.x % L * 8;
    const int64_t step = (int64_t)gridDim.x * (NT / L), first = (int64_t)blockIdx.x * (NT / L);
    float post_w[8], post_b[8], pre_w[8], pre_b[8], scale[8];
    auto params = [&] {
        load_columns<kEven>(s.post_w, s.width, col, 1.f, post_w);
        load_columns<kEven>(s.post_b, s.width, col, 0.f, post_b);
        load_columns<kEven>(s.pre_w, s.width, col, 1.f, pre_w);
        load_columns<kEven>(s.pre_b, s.width, col, 0.f, pre_b);
        load_columns<kEven>(s.scale, s.width, col, s.factor, scale);
    };
    Raw8<T> nx, nf;
    auto load = [&](int64_t r0) {
        const int64_t row = r0 + threadIdx.x / L;
        const bool ok = row < s.rows;
        nx = load_row<T, kEven>(ok ? a.x + row * s.width : nullptr, s.width, col);
        nf = load_row<T, kEven>(ok && a.f ? a.f + row * s.width : nullptr, s.width, col);
    };
    if (kAhead) {
        params();
        load(first);
    }
    for (int64_t r0 = first; r0 < s.rows; r0 += step) {
        const int64_t row = r0 + threadIdx.x / L, at = row * s.width + col;
        const bool ok = row < s.rows && col < s.width;
        float x[8], f[8], w[8];
        if (!kAhead) load(r0);
        row_values<T>(nx, x);
        row_values<T>(nf, f);
        if (kAhead && r0 + step < s.rows) load(r0 + step);
        if (!kAhead) params();
        if (s.post) {
            unit_row<kRms>(f, row < s.rows ? s.eps : 1.f, s.width, col, sums);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = fmaf(f[i], post_w[i], post_b[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = scale[i];
        if (a.gate) {
            float g[8];
            row_values<T>(load_row<T, kEven>(row < s.rows ? a.gate + row / s.gate_rows * s.width : nullptr, s.width, col), g);
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] *= g[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fmaf(w[i], f[i], x[i]);
        if (ok && a.y) store8<T>(a.y + at, x, kEven ? 8 : s.width - col);
        if (s.pre) {
            unit_row<kRms>(x, row < s.rows ? s.eps : 1.f, s.width, col, sums);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i], pre_w[i], pre_b[i]);
            if (ok) store8<T>(a.u + at, x, kEven ? 8 : s.width - col);
        }
    }
}

// sums acc over the row groups of the workgroup and hands out one row of width values
template <int L, int NT, class F>
__device__ __forceinline__ void group_columns(const float (&acc)[8], float* lds, int width, F put) {
    const int col = threadIdx.x % L * 8;
    if constexpr (NT == L) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < width) put(col + i, acc[i]);
    } else {
        constexpr int kCols = L * 8;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) lds[threadIdx.x / L * kCols + col + i] = acc[i];
        __syncthreads();
        for (int c = threadIdx.x; c < width; c += NT) {
            float v = 0.f;
            for (int q = 0; q < NT / L; ++q) v += lds[q * kCols + c];
            put(c, v);
        }
    }
}

template <int T, int L, int NT, bool kRms, bool kEven>
__global__ __launch_bounds__(NT) void norm_bwd_kernel(NormArgs<T> a) {
    constexpr int G = NT / L;
    constexpr bool kAhead = NT < 1024;
    const NormShape& s = a.s;
    __shared__ float lds[4 * (NT / 64)];
    __shared__ float cols[G > 1 ? G * L * 8 : 1];
    RowSums<L, NT> sums = {lds, 0};
    const int col = threadIdx.x % L * 8;
    float post_w[8], post_b[8], pre_w[8], scale[8], gate[8];
    float s_prew[8], s_preb[8], s_postw[8], s_postb[8], s_scale[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { s_prew[i] = s_preb[i] = s_postw[i] = s_postb[i] = s_scale[i] = 0.f; gate[i] = 1.f; }
    auto params = [&] {
        load_columns<kEven>(s.post_w, s.width, col, 1.f, post_w);
        load_columns<kEven>(s.post_b, s.width, col, 0.f, post_b);
        load_columns<kEven>(s.pre_w, s.width, col, 1.f, pre_w);
        load_columns<kEven>(s.scale, s.width, col, s.factor, scale);
    };
    if (kAhead) params();
    for (int64_t unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        const int64_t gate_row = unit / a.cuts, first = gate_row * s.gate_rows + (unit - gate_row * a.cuts) * a.unit_rows;
        const int64_t group_end = (gate_row + 1) * s.gate_rows, end0 = first + a.unit_rows, end = end0 < group_end ? end0 : group_end;
        float s_z[8];                         // sum of grad_y_total * z: the gate's gradient up to the scale, the scale's up to the gate
#pragma unroll
        for (int i = 0; i < 8; ++i) s_z[i] = 0.f;
        if (a.gate) row_values<T>(load_row<T, kEven>(a.gate + gate_row * s.width, s.width, col), gate);
        Raw8<T> nx, nf, ngy, ngu;
        auto load = [&](int64_t r0) {
            const int64_t row = r0 + threadIdx.x / L, at = row * s.width;
            const bool ok = row < end;
            nf = load_row<T, kEven>(ok && a.f ? a.f + at : nullptr, s.width, col);
            nx = load_row<T, kEven>(ok ? a.x + at : nullptr, s.width, col);
            ngu = load_row<T, kEven>(ok && a.gu ? a.gu + at : nullptr, s.width, col);
            ngy = load_row<T, kEven>(ok && a.gy ? a.gy + at : nullptr, s.width, col);
        };
        if (kAhead) load(first);
        for (int64_t r0 = first; r0 < end; r0 += G) {
            const int64_t row = r0 + threadIdx.x / L, at = row * s.width + col;
            const bool ok = row < end && col < s.width;
            const float eps = row < end ? s.eps : 1.f;      // rows behind the run are zeros: without a spread, eps = 0 would make them NaN in the sums
            float x[8], f[8], gy[8], gu[8], z[8], fr = 1.f;
            if (!kAhead) load(r0);
            row_values<T>(nf, f);
            row_values<T>(nx, x);
            row_values<T>(ngu, gu);
            row_values<T>(ngy, gy);
            if (kAhead && r0 + G < end) load(r0 + G);
            if (!kAhead) params();
            if (s.post) {
                fr = unit_row<kRms>(f, eps, s.width, col, sums);
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = fmaf(f[i], post_w[i], post_b[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = f[i];
            }
            if (s.pre) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = fmaf(scale[i] * gate[i], z[i], x[i]);
                const float yr = unit_row<kRms>(x, eps, s.width, col, sums);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    s_prew[i] = fmaf(gu[i], x[i], s_prew[i]);
                    if (!kRms || s.pre_b) s_preb[i] += gu[i];
                    gu[i] *= pre_w[i];
                }
                unit_row_grad<kRms>(gu, x, yr, s.width, col, sums);
#pragma unroll
                for (int i = 0; i < 8; ++i) gy[i] += gu[i];
            }
            if (ok && a.gx) store8<T>(a.gx + at, gy, kEven ? 8 : s.width - col);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s_z[i] = fmaf(gy[i], z[i], s_z[i]);
                gy[i] *= scale[i] * gate[i];
            }
            if (s.post) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    s_postw[i] = fmaf(gy[i], f[i], s_postw[i]);
                    if (!kRms || s.post_b) s_postb[i] += gy[i];
                    gy[i] *= post_w[i];
                }
                if (a.gf) unit_row_grad<kRms>(gy, f, fr, s.width, col, sums);
            }
            if (ok && a.gf) store8<T>(a.gf + at, gy, kEven ? 8 : s.width - col);
        }
        if (!kAhead) params();
#pragma unroll
        for (int i = 0; i < 8; ++i) s_scale[i] = fmaf(s_z[i], gate[i], s_scale[i]);
        if (a.want & 32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s_z[i] *= scale[i];
            if (a.cuts == 1) group_columns<L, NT>(s_z, cols, s.width, [&](int c, float v) { store_value<T>(a.ggate + gate_row * s.width + c, v); });
            else group_columns<L, NT>(s_z, cols, s.width, [&](int c, float v) { a.gate_part[unit * s.width + c] = v; });
        }
    }
    auto put = [&](int k, const float (&acc)[8]) {
        if (a.want >> k & 1)
            group_columns<L, NT>(acc, cols, s.width, [&](int c, float v) { a.part[((int64_t)k * gridDim.x + blockIdx.x) * s.width + c] = v; });
    };
    put(0, s_prew);
    put(1, s_preb);
    put(2, s_postw);
    put(3, s_postb);
    put(4, s_scale);
}

struct NormColumns { float* out[5]; };

// The parameters' gradients (blockIdx.y 0..4: sums of the workgroups' partial rows) and the gate's (from 5 on: a gate row from its cuts),
// in order: 16 columns x 16 runs of rows per workgroup, the runs joined in LDS.
template <int T>
__global__ __launch_bounds__(256) void norm_columns_kernel(const float* part, int parts, const float* gate_part, int cuts, int width, NormColumns o,
                                                           typename Num<T>::type* ggate) {
    __shared__ float lds[16][17];
    const int k = blockIdx.y, c = blockIdx.x * 16 + (threadIdx.x & 15), q = threadIdx.x >> 4;
    if (k < 5 && !o.out[k]) return;
    const int n = k < 5 ? parts : cuts;
    const float* p = (k < 5 ? part + (int64_t)k * parts * width : gate_part + (int64_t)(k - 5) * cuts * width) + c;
    float v = 0.f;
    if (c < width)
#pragma unroll 8
        for (int i = q; i < n; i += 16) v += p[(int64_t)i * width];
    lds[q][threadIdx.x & 15] = v;
    __syncthreads();
    if (threadIdx.x >= 16 || c >= width) return;
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) v += lds[i][threadIdx.x];
    if (k < 5) o.out[k][c] = v;
    else store_value<T>(ggate + (int64_t)(k - 5) * width + c, v);
}

// threads of a row and of a workgroup by the width: the row fits the registers, narrow rows share a wave
static int norm_group_rows(int width) { return width <= 64 ? 32 : width <= 512 ? 4 : 1; }

struct NormPlan { int64_t units; int unit_rows, cuts, blocks; };
// Backward: up to 768 workgroups (three per compute unit).  With a gate, a unit is a run of rows of one gate row (a gate row with many
// rows is cut); without, a run of rows.
static NormPlan norm_plan(const NormShape& s, bool gated) {
    NormPlan p;
    const int g = norm_group_rows(s.width);
    const int64_t groups = s.rows / s.gate_rows, most = 768;
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
#define EQ_NORM_EVEN(L, NT, EVEN)                                                                       \
    do {                                                                                                \
        if (backward && a.s.rms) norm_bwd_kernel<T, L, NT, true, EVEN><<<blocks, NT, 0, st>>>(a);       \
        else if (backward) norm_bwd_kernel<T, L, NT, false, EVEN><<<blocks, NT, 0, st>>>(a);            \
        else if (a.s.rms) norm_fwd_kernel<T, L, NT, true, EVEN><<<blocks, NT, 0, st>>>(a);              \
        else norm_fwd_kernel<T, L, NT, false, EVEN><<<blocks, NT, 0, st>>>(a);                          \
    } while (0)
#define EQ_NORM(L, NT)                       \
    do {                                     \
        if (w % 8 == 0) EQ_NORM_EVEN(L, NT, true); \
        else EQ_NORM_EVEN(L, NT, false);     \
    } while (0)
    if (w <= 64) EQ_NORM(8, 256);
    else if (w <= 512) EQ_NORM(64, 256);
    else if (w <= 2048) EQ_NORM(256, 256);
    else if (w <= 4096) EQ_NORM(512, 512);
    else EQ_NORM(1024, 1024);
#undef EQ_NORM
#undef EQ_NORM_EVEN
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
    EQ_CHECK_ARG(d->rows == 0 || d->f || (d->pre_weight && !d->gate && !d->scale && !d->post_weight), EQUIGSPR_EINVAL,
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
    return norm_run<T>(a, false, (int)(groups < 2048 ? groups : 2048), st);
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
    const bool gate_cut = a.ggate && p.cuts > 1;
    if (columns || gate_cut) {
        norm_columns_kernel<T><<<dim3(ceil_div(s.width, 16), 5 + (gate_cut ? (unsigned)(s.rows / s.gate_rows) : 0)), 256, 0, st>>>(
            a.part, p.blocks, a.gate_part, p.cuts, s.width, c, a.ggate);
        EQ_CHECK_LAUNCH("residual_norm_backward (columns)");
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
