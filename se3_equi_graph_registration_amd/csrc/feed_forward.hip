// The gated feed-forward block:  z = x Wg^T + bg,  u = x Wu^T + bu,  h = act(z) * u,  y = h Wd^T + bd,  and its backward
//   dh = dy Wd,  dz = dh u act'(z),  du = dh act(z),  dx = dz Wg + du Wu,  dWg = dz^T x,  dWu = du^T x,  dWd = dy^T h,  biases: column sums.
// One matrix-product kernel, three epilogues:
//   kGate   both projections of a tile from one staged x tile, activation and product in registers: h (and, for training, z | u) leave once
//   kGrad   dh of a tile never leaves: the epilogue reads z | u and writes dz | du
//   kPlain  C = A B^T (+ bias), or fp32 partial tiles of a cut contraction, summed in order by ff_sum_kernel
// z | u and dz | du are [rows, 2 hidden]: dx is ONE product over 2 hidden, dWg and dWu are the two halves of ONE product's rows.
// A product's operands may run along or across the contraction in memory; across, the tile is read transposed (planes.h), so nothing
// is ever transposed in memory.  Products accumulate in fp32.  h, dz and du are operands of further products and are stored in the
// inputs' type (one rounding each); z | u, which only the epilogue of the backward reads, stays fp32 -- in 16 bits its rounding would come
// on top of dz's and du's in every gradient (bf16: 1.8 instead of 1.4 times the outputs' own rounding).
// fp16: dz and du are held as 2^E dz and 2^E du, with E from the largest |dy| (ff_held), undone in fp32 where their products leave.
// Bound: for many rows the matrix pipe together with what does not run beside it -- it is busy 0.43..0.51 of the time in the plain products, 0.33
// in the projections and 0.19 in the hidden gradients, whose epilogues (0.7 and 0.8 GB) run alone, one workgroup per compute unit; for few
// rows the weights' bytes.  Measured, bf16, 16384 x 1024 x 4096: projections 402 us (685 TFLOP/s,
// with 0.7 GB of results), output 147 (935), hidden gradients 330 (415, with 0.8 GB through its epilogue), input 276 (995), weights 300 + 161 (915, 855).
#include "planes.h"

#include <math.h>

namespace eq {

enum { kPlain = 0, kGate = 1, kGrad = 2 };
enum { kSilu = EQUIGSPR_ACT_SILU, kGelu = EQUIGSPR_ACT_GELU, kRelu = EQUIGSPR_ACT_RELU };

// one operand as rows of `len` values; row r lies at p + r * ld, rows at or behind `split` in q (two matrices that act as one)
template <int T>
struct FfOperand {
    const typename Num<T>::type *p, *q;
    int64_t ld;
    int rows, split, len;
    __device__ __forceinline__ const typename Num<T>::type* row(int r) const { return r < split ? p + r * ld : q + (r - split) * ld; }
};

template <int T>
struct FfArgs {
    using E = typename Num<T>::type;
    FfOperand<T> a, b;                        // the output's rows and columns
    int m, n, k;                              // kGate: n counts the columns of one projection
    int tiles_m, tiles_n, cuts, cut_k;        // cut_k: contraction length of a cut (a multiple of the k tile)
    E* c;                                     // [m, n]
    const E *bias, *bias2;
    float* part;                              // [cuts][m][n]
    float* zu;                                // kGate: written if not null; kGrad: read.  [m, 2 n]
    E* dzu;                                   // kGrad: [m, 2 n]
    const float* range;                       // fp16 backward: [kFfRange], largest |dy|; kGrad scales dz | du by ff_held, kPlain divides by it.  Null: 1
    int act;
};

__device__ __forceinline__ void floats_of(const Raw8<kF32>& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = raw_float<kF32>(r, i);
}

// fp16: the power of two that dz and du are held with, so that output gradients far below 1 do not sink into fp16's smallest steps and
// far larger ones do not leave its range.  1 while the largest |dy| lies in [2^-4, 2^4); otherwise it brings that to [2^-4, 2^-3) or [2^3, 2^4):
// dz and du may then be 2^12 times it, and keep all their bits down to 2^-10 of it.
constexpr int kFfRange = 256;                 // workgroups that look for the largest |dy|
template <int T>
__device__ __forceinline__ float ff_held(const float* range) {
    if constexpr (T != kF16) return 1.f;
    if (!range) return 1.f;
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < kFfRange / 64; ++i) m = fmaxf(m, range[(threadIdx.x & 63) + 64 * i]);
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (!(m > 0.f) || m == INFINITY) return 1.f;
    const int e = ilogbf(m);
    return ldexpf(1.f, e < -4 ? -4 - e : e >= 4 ? 3 - e : 0);
}
template <int T>
__global__ __launch_bounds__(1024) void ff_range_kernel(const typename Num<T>::type* x, int64_t n, float* range) {
    float m = 0.f;
    for (int64_t i = ((int64_t)blockIdx.x * 1024 + threadIdx.x) * 8; i < n; i += (int64_t)kFfRange * 1024 * 8) {
        float v[8];
        load8f<T>(x + i, n - i < 8 ? (int)(n - i) : 8, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]));
    }
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    __shared__ float part[16];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) m = fmaxf(m, part[i]);
    range[blockIdx.x] = m;
}

// act(z) and its derivative
__device__ __forceinline__ void activate(int act, float z, float& a, float& d) {
    if (act == kSilu) {
        const float s = 1.f / (1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
        a = z * s;
        d = s * (1.f + z * (1.f - s));
    } else if (act == kGelu) {
        const float c = 0.5f * (1.f + erff(z * 0.70710678118654752f));
        a = z * c;
        d = fmaf(z * 0.39894228040143268f, __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z), c);
    } else {                                      // NaN stays NaN in both
        a = z <= 0.f ? 0.f : z;
        d = z > 0.f ? 1.f : z <= 0.f ? 0.f : z;
    }
}

// Two output tiles.  Large: 256 x 256, eight waves of 128 x 64, two buffers of 64 k (16-bit types): per step of 16 a wave reads six
// operands for eight products, a compute unit's LDS keeps up with its matrix pipes, and memory is read half as often as by 128 x 128.
// Small: 128 x 128, four waves of 64 x 64, one buffer; for outputs that would leave compute units idle, and for the three planes of fp32.
template <int T, bool kLarge>
struct FfShapeOf {
    static_assert(!kLarge || T != kF32, "three planes do not fit the large tile");
    static constexpr int kBK = T == kF32 ? 32 : 64, kMB = kLarge ? 4 : 2, kWavesN = kLarge ? 4 : 2, kWaves = 2 * kWavesN;
    static constexpr int kBM = 2 * kMB * 32, kBN = kWavesN * 64, kThreads = kWaves * 64, kBuffers = kLarge ? 2 : 1;
};

// kAcross: the operand's contraction runs across its rows in memory (tile [k][outer]) instead of along them (tile [outer][k])
template <int T, bool kAcross, int kOuter, int BK, int NT>
struct FfTile {
    using E = typename Num<T>::type;
    static constexpr int W = kAcross ? kOuter : BK, ROWS = kAcross ? BK : kOuter;
    static constexpr int kPlane = Tile<W>::size(ROWS), kPer = ROWS * W / 8 / NT;
    static_assert(kPer * NT * 8 == ROWS * W, "whole chunks per thread");
    Raw8<T> raw[kPer];
    // outer0: first output row / column of the tile; k0: first contraction index; k_end bounds it.  outer_row(r, clamp): the memory row of
    // output r (along): null where there is none, or the last one if clamp (its products are never stored)
    template <class F>
    __device__ __forceinline__ void load(const FfOperand<T>& o, int outer0, int k0, int k_end, F outer_row) {
        const bool whole = k0 + BK <= k_end && (!kAcross || o.len % 8 == 0 || outer0 + W <= o.len);      // no chunk is cut
        if (whole) {
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
                const int id = threadIdx.x + u * NT, r = id / (W / 8), c = id % (W / 8) * 8;
                if constexpr (kAcross) {
                    if (outer0 + c < o.len) raw[u] = load8<T>(o.row(k0 + r) + outer0 + c, 0, 8);
                    else raw[u] = raw_zero<T>();
                } else {
                    raw[u] = load8<T>(outer_row(r, true) + k0 + c, 0, 8);
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
                const int id = threadIdx.x + u * NT, r = id / (W / 8), c = id % (W / 8) * 8;
                const auto cut = [](const E* from, int at, int width) { return NT == 512 ? load8_small<T>(from, at, width) : load8<T>(from, at, width); };
                if constexpr (kAcross) {
                    raw[u] = k0 + r < k_end ? cut(o.row(k0 + r) + outer0, c, o.len - outer0) : raw_zero<T>();
                } else {
                    const E* row = outer_row(r, false);
                    raw[u] = row ? cut(row + k0, c, k_end - k0) : raw_zero<T>();
                }
            }
        }
    }
    __device__ __forceinline__ void store(short* tile) const {
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            const int id = threadIdx.x + u * NT;
            const Op8<T> o = planes_of<T>(raw[u]);
#pragma unroll
            for (int p = 0; p < Num<T>::planes; ++p) *reinterpret_cast<s16x8*>(tile + p * kPlane + Tile<W>::at(id / (W / 8), id % (W / 8))) = o.p[p];
        }
    }
    // 32 outputs from o0, k-step ks
    __device__ static __forceinline__ Op8<T> operand(const short* tile, int o0, int ks, int lane) {
        Op8<T> r;
#pragma unroll
        for (int p = 0; p < Num<T>::planes; ++p) {
            const short* t = tile + p * kPlane;
            if constexpr (kAcross) {
                const int k = 16 * ks + 8 * (lane >> 5), c = o0 + (lane & 16);
                r.p[p] = join8(Tile<W>::col4(t, k, c, lane), Tile<W>::col4(t, k + 4, c, lane));
            } else {
                r.p[p] = Tile<W>::row8(t, o0 + (lane & 31), 2 * ks + (lane >> 5));
            }
        }
        return r;
    }
};

template <int T, bool kAcrossA, bool kAcrossB, int kEpi, bool kLarge>
__global__ __launch_bounds__((FfShapeOf<T, kLarge>::kThreads), 2) void ff_product_kernel(FfArgs<T> g) {
    using S = FfShapeOf<T, kLarge>;
    using E = typename Num<T>::type;
    constexpr int BK = S::kBK, BM = S::kBM, BN = S::kBN, MB = S::kMB, NP = Num<T>::planes, TN = kEpi == kGate ? BN / 2 : BN, NBUF = S::kBuffers;
    using TA = FfTile<T, kAcrossA, BM, BK, S::kThreads>;
    using TB = FfTile<T, kAcrossB, BN, BK, S::kThreads>;
    // the staged tiles; at the end each wave turns 32 x 64 results at a time from matrix layout to rows in its own part
    constexpr int kTileA = NP * TA::kPlane, kTileB = NP * TB::kPlane, kOutStride = 68, kOutFloats = 32 * kOutStride;
    __shared__ __attribute__((aligned(16))) short lds[NBUF * (kTileA + kTileB)];
    static_assert(sizeof(lds) >= sizeof(float) * kOutFloats * S::kWaves, "room for the results");
    auto tile_a = [&](int buf) { return lds + buf * kTileA; };
    auto tile_b = [&](int buf) { return lds + NBUF * kTileA + buf * kTileB; };
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, wm = wave / S::kWavesN, wn = wave % S::kWavesN;
    // neighbours on an XCD take 8 row tiles by some column tiles: both operands' panels are shared in its L2
    const int id = xcd_block(blockIdx.x, gridDim.x), per_cut = g.tiles_m * g.tiles_n, cut = id / per_cut, rest = id - cut * per_cut;
    const int band = rest / (8 * g.tiles_n), in_band = rest - band * 8 * g.tiles_n, band_rows = min(8, g.tiles_m - 8 * band);
    const int tm = 8 * band + in_band % band_rows, tn = in_band / band_rows;
    const int m0 = tm * BM, n0 = tn * TN, k_begin = cut * g.cut_k, k_end = min(g.k, k_begin + g.cut_k);
    auto row_a = [&](int r, bool clamp) -> const E* {
        const int m = m0 + r;
        return clamp ? g.a.row(min(m, g.a.rows - 1)) : m < g.a.rows ? g.a.row(m) : nullptr;
    };
    auto row_b = [&](int r, bool clamp) -> const E* {
        if constexpr (kEpi == kGate) {            // the tile's first half: columns of one projection; its second half: the same of the other
            int c = n0 + r % TN;
            if (clamp) c = min(c, g.n - 1);
            return c < g.n ? (r < TN ? g.b.p : g.b.q) + c * g.b.ld : nullptr;
        } else {
            const int n = n0 + r;
            return clamp ? g.b.row(min(n, g.b.rows - 1)) : n < g.b.rows ? g.b.row(n) : nullptr;
        }
    };
    // acc[i][j]: C tile with the output's columns in the registers (block j) and its rows in the lanes (block i)
    pf32x16 acc[MB][2];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    const int om = wm * MB * 32;
    const int on[2] = {kEpi == kGate ? wn * 32 : wn * 64, kEpi == kGate ? TN + wn * 32 : wn * 64 + 32};
    TA sa;
    TB sb;
    // Operands are fetched one step of 16 ahead of their products (two sets of registers): the fence between keeps the compiler from
    // sinking the reads to their uses, where their latency would be paid at every step.
    Op8<T> pa[2][MB], pb[2][2];
    constexpr int KS = BK / 16;
    auto fetch = [&](int buf, int ks, int set) {
#pragma unroll
        for (int j = 0; j < 2; ++j) pb[set][j] = TB::operand(tile_b(buf), on[j], ks, lane);
#pragma unroll
        for (int i = 0; i < MB; ++i) pa[set][i] = TA::operand(tile_a(buf), om + 32 * i, ks, lane);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto products = [&](int set) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) mma<T>(acc[i][j], pb[set][j], pa[set][i]);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto load = [&](int k0) {
        sa.load(g.a, m0, k0, k_end, row_a);
        sb.load(g.b, n0, k0, k_end, row_b);
    };
    auto store = [&](int buf) {
        sa.store(tile_a(buf));
        sb.store(tile_b(buf));
    };
    load(k_begin);
    if constexpr (NBUF == 2) {
        // One meeting of the waves per tile, before its last products: the next tile, written halfway, is then readable while those run,
        // and its memory loads were issued a whole tile earlier.
        static_assert(KS % 2 == 0, "the next tile starts in the first register set");
        store(0);
        if (k_begin + BK < k_end) load(k_begin + BK);
        __syncthreads();
        fetch(0, 0, 0);
        int buf = 0;
        for (int k0 = k_begin; k0 < k_end; k0 += BK, buf ^= 1) {
            const bool more = k0 + BK < k_end;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (ks + 1 < KS) fetch(buf, ks + 1, (ks + 1) & 1);
                if (ks == KS / 2 && more) {
                    store(buf ^ 1);
                    if (k0 + 2 * BK < k_end) load(k0 + 2 * BK);
                }
                if (ks + 1 == KS && more) {
                    __syncthreads();
                    fetch(buf ^ 1, 0, 0);
                }
                products(ks & 1);
            }
        }
    } else {
        for (int k0 = k_begin; k0 < k_end; k0 += BK) {
            __syncthreads();
            store(0);
            __syncthreads();
            if (k0 + BK < k_end) load(k0 + BK);
            fetch(0, 0, 0);
            if constexpr (T == kF32) {
                // The twelve products of a k tile in an accumulator of their own, added by the vector ALU: the matrix pipe does not round
                // to nearest when it adds to a large accumulator, and what that leaves adds up in sums over rows (biases' gradients).
                static_assert(KS == 2, "both steps' operands are held at once");
                fetch(0, 1, 1);
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        pf32x16 t;
#pragma unroll
                        for (int r = 0; r < 16; ++r) t[r] = 0.f;
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks) mma<T>(t, pb[ks][j], pa[ks][i]);
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[i][j][r] += t[r];
                    }
            } else {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    if (ks + 1 < KS) fetch(0, ks + 1, (ks + 1) & 1);
                    products(ks & 1);
                }
            }
        }
    }
    __syncthreads();                              // the last tiles have been read
    const float held = kEpi == kGate ? 1.f : ff_held<T>(g.range), back = 1.f / held;
    float* const out = reinterpret_cast<float*>(lds) + wave * kOutFloats;
    constexpr int kCols = kEpi == kGate ? 32 : 64, kLanes = kCols / 8, kRows = 64 / kLanes;      // columns, lanes per row, rows of a step
    const int col = n0 + (kEpi == kGate ? wn * 32 : wn * 64) + lane % kLanes * 8, left = g.n - col;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<pf32x4*>(out + (lane & 31) * kOutStride + 32 * j + 8 * q + 4 * half) =
                    (pf32x4){acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        // kGrad, small tile: what the epilogue reads from memory is requested for all of this block's steps before the first one needs it
        // (few workgroups, nothing else hides the latency; the large tile has no registers for it and its own neighbours to hide it)
        constexpr bool kAll = kEpi == kGrad && !kLarge;
        Raw8<kF32> pz[kAll ? 32 / kRows : 1], pu[kAll ? 32 / kRows : 1];
        if constexpr (kAll) {
#pragma unroll
            for (int p = 0; p < 32 / kRows; ++p) {
                const float* src = g.zu + (int64_t)min(m0 + om + 32 * i + p * kRows + lane / kLanes, g.m - 1) * 2 * g.n;
                pz[p] = left > 0 ? load8<kF32>(src, col, g.n) : raw_zero<kF32>();
                pu[p] = left > 0 ? load8<kF32>(src + g.n, col, g.n) : raw_zero<kF32>();
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll(kAll ? 4 : 1)
        for (int r0 = 0; r0 < 32; r0 += kRows) {
            const int r = r0 + lane / kLanes, row = m0 + om + 32 * i + r;
            float v[8], z[8], u[8];
            const float* src = out + r * kOutStride + lane % kLanes * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = src[e];
            if (row >= g.m || left <= 0) continue;
            if constexpr (kEpi == kGate) {
                float h[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) { z[e] = 0.f; u[e] = 0.f; }
                if (g.bias) load8f<T>(g.bias + col, left, z);
                if (g.bias2) load8f<T>(g.bias2 + col, left, u);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float a, d;
                    z[e] += v[e];
                    u[e] += src[32 + e];
                    activate(g.act, z[e], a, d);
                    h[e] = a * u[e];
                }
                store8<T>(g.c + (int64_t)row * g.n + col, h, left);
                if (g.zu) {
                    store8<kF32>(g.zu + (int64_t)row * 2 * g.n + col, z, left);
                    store8<kF32>(g.zu + (int64_t)row * 2 * g.n + g.n + col, u, left);
                }
            } else if constexpr (kEpi == kGrad) {
                const int64_t at = (int64_t)row * 2 * g.n + col;
                if constexpr (kAll) {
                    floats_of(pz[r0 / kRows], z);
                    floats_of(pu[r0 / kRows], u);
                } else {
                    load8f<kF32>(g.zu + at, left, z);
                    load8f<kF32>(g.zu + at + g.n, left, u);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float a, d;
                    activate(g.act, z[e], a, d);
                    if constexpr (T == kF16) v[e] *= held;
                    z[e] = v[e] * u[e] * d;
                    u[e] = v[e] * a;
                }
                store8<T>(g.dzu + at, z, left);
                store8<T>(g.dzu + at + g.n, u, left);
            } else if (g.cuts > 1) {
                store8<kF32>(g.part + ((int64_t)cut * g.m + row) * g.n + col, v, left);
            } else {
                if constexpr (T == kF16) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= back;
                }
                if (g.bias) {
                    load8f<T>(g.bias + col, left, z);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += z[e];
                }
                store8<T>(g.c + (int64_t)row * g.n + col, v, left);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// Few rows (single tokens): the weights' bytes are the work.  A workgroup owns 16 output columns, its eight waves share out the contraction;
// a lane streams 16 bytes of one weight row at a time straight into the A operand of v_mfma_f32_16x16x32 (four lanes 64 consecutive bytes),
// the rows are the B operand, read from the caches, and the waves' sums meet in LDS in order.  Measured in bf16 at 8 x 2048 x 5632:
// projections 14 us (3.4 TB/s; 29 by tiles), output 10 (2.3 TB/s; 13).
template <int T>
__device__ __forceinline__ void mma16(pf32x4& acc, const Op8<T>& a, const Op8<T>& b) {
    auto one = [&](s16x8 x, s16x8 y) {
        if constexpr (T == kF16) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pf16x8, x), __builtin_bit_cast(pf16x8, y), acc, 0, 0, 0);
        else acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pbf16x8, x), __builtin_bit_cast(pbf16x8, y), acc, 0, 0, 0);
    };
    if constexpr (T == kF32) {
        one(a.p[2], b.p[0]);
        one(a.p[0], b.p[2]);
        one(a.p[1], b.p[1]);
        one(a.p[1], b.p[0]);
        one(a.p[0], b.p[1]);
    }
    one(a.p[0], b.p[0]);
}

constexpr int kFewWaves = 8, kFewStep = 128;
// RB: blocks of 16 rows
template <int T, int RB, int kEpi>
__global__ __launch_bounds__(kFewWaves * 64) void ff_few_kernel(FfArgs<T> g) {
    using E = typename Num<T>::type;
    constexpr int NM = kEpi == kGate ? 2 : 1;             // weight matrices
    __shared__ __attribute__((aligned(16))) float sums[kFewWaves][NM][RB][64][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, grp = lane >> 4, n0 = blockIdx.x * 16;
    const int k_begin = wave * g.cut_k, k_end = min(g.k, k_begin + g.cut_k);
    const int n = min(n0 + (lane & 15), g.n - 1);         // rows behind the last: its copies, never stored
    const E* w[2] = {g.b.p + n * g.b.ld, g.b.q + n * g.b.ld};
    const E* x[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) x[r] = g.a.p + min(16 * r + (lane & 15), g.m - 1) * g.a.ld;
    pf32x4 acc[NM][RB];
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int r = 0; r < RB; ++r) acc[i][r] = (pf32x4){0.f, 0.f, 0.f, 0.f};
    auto step = [&](int k0, auto load) {
        Raw8<T> rw[NM][4], rx[RB][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = k0 + 32 * i + 8 * grp;
#pragma unroll
            for (int j = 0; j < NM; ++j) rw[j][i] = load(w[j], k);
#pragma unroll
            for (int r = 0; r < RB; ++r) rx[r][i] = load(x[r], k);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            Op8<T> ox[RB];
#pragma unroll
            for (int r = 0; r < RB; ++r) ox[r] = planes_of<T>(rx[r][i]);
#pragma unroll
            for (int j = 0; j < NM; ++j) {
                const Op8<T> ow = planes_of<T>(rw[j][i]);
#pragma unroll
                for (int r = 0; r < RB; ++r) mma16<T>(acc[j][r], ow, ox[r]);
            }
        }
    };
    int k0 = k_begin;
#pragma unroll 2
    for (; k0 + kFewStep <= k_end; k0 += kFewStep) step(k0, [&](const E* p, int k) { return load8<T>(p + k, 0, 8); });
    if (k0 < k_end) step(k0, [&](const E* p, int k) { return k < k_end ? load8<T>(p + k, 0, k_end - k) : raw_zero<T>(); });
#pragma unroll
    for (int j = 0; j < NM; ++j)
#pragma unroll
        for (int r = 0; r < RB; ++r) *reinterpret_cast<pf32x4*>(sums[wave][j][r][lane]) = acc[j][r];
    __syncthreads();
    if (wave >= RB) return;                               // wave r finishes row block r: lane = row, four consecutive columns
    const int row = 16 * wave + (lane & 15), col = n0 + 4 * grp, left = g.n - col;
    if (row >= g.m || left <= 0) return;
    float v[NM][4];
#pragma unroll
    for (int j = 0; j < NM; ++j) {
        const E* bias = j ? g.bias2 : g.bias;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j][e] = 0.f;
        if (bias) load4<T>(bias + col, left, v[j]);
        for (int q = 0; q < kFewWaves; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] += sums[q][j][wave][lane][e];
    }
    if constexpr (kEpi == kGate) {
        float h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float a, d;
            activate(g.act, v[0][e], a, d);
            h[e] = a * v[1][e];
        }
        store4<T>(g.c + (int64_t)row * g.n + col, h, left);
        if (g.zu) {
            store4<kF32>(g.zu + (int64_t)row * 2 * g.n + col, v[0], left);
            store4<kF32>(g.zu + (int64_t)row * 2 * g.n + g.n + col, v[1], left);
        }
    } else {
        store4<T>(g.c + (int64_t)row * g.n + col, v[0], left);
    }
}

// the parts of a cut contraction, in order
template <int T>
__global__ __launch_bounds__(256) void ff_sum_kernel(FfArgs<T> g) {
    const int64_t n = (int64_t)g.m * g.n;
    const float back = 1.f / ff_held<T>(g.range);      // 1 wherever there is a bias
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float v = g.bias ? (float)g.bias[i % g.n] : 0.f;
#pragma unroll 8
        for (int c = 0; c < g.cuts; ++c) v += g.part[c * n + i];
        if constexpr (T == kF16) v *= back;
        store_value<T>(g.c + i, v);
    }
}

// The biases' gradients: column sums of dz | du and of dy in one launch, by runs of rows, then the runs in order.  A workgroup takes 64
// columns of a run, 4 rows at a time.
template <int T>
struct FfColumns {
    const typename Num<T>::type* x[2];
    typename Num<T>::type* out[2];
    int width[2];                             // 0: not wanted
    int rows, runs;
    const float* range;                       // fp16: as FfArgs::range, for x[0]
};
constexpr int kFfRun = 128;                   // rows of a run
template <int T>
__global__ __launch_bounds__(256) void ff_columns_kernel(FfColumns<T> a, float* part) {
    const int first = (a.width[0] + 63) / 64, which = (int)blockIdx.x >= first, block0 = which ? first : 0;
    const int width = a.width[which], c = ((int)blockIdx.x - block0) * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
    const int r0 = blockIdx.y * kFfRun, r1 = min(a.rows, r0 + kFfRun);
    __shared__ float lds[4][64];
    float v = 0.f;
    if (c < width) {
        const typename Num<T>::type* x = a.x[which] + c;
#pragma unroll 8
        for (int r = r0 + q; r < r1; r += 4) v += (float)x[(int64_t)r * width];
    }
    lds[q][threadIdx.x & 63] = v;
    __syncthreads();
    if (q == 0 && c < width)
        part[(int64_t)blockIdx.y * (a.width[0] + a.width[1]) + (which ? a.width[0] : 0) + c] =
            (lds[0][threadIdx.x] + lds[1][threadIdx.x]) + (lds[2][threadIdx.x] + lds[3][threadIdx.x]);
}
template <int T>
__global__ __launch_bounds__(256) void ff_columns_sum_kernel(FfColumns<T> a, const float* part) {
    const int all = a.width[0] + a.width[1], c = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
    __shared__ float lds[4][64];
    const float back = 1.f / ff_held<T>(a.range);
    float v = 0.f;
    if (c < all)
#pragma unroll 8
        for (int r = q; r < a.runs; r += 4) v += part[(int64_t)r * all + c];
    lds[q][threadIdx.x & 63] = v;
    __syncthreads();
    if (q || c >= all) return;
    v = (lds[0][threadIdx.x] + lds[1][threadIdx.x]) + (lds[2][threadIdx.x] + lds[3][threadIdx.x]);
    if (c < a.width[0]) store_value<T>(a.out[0] + c, T == kF16 ? v * back : v);
    else store_value<T>(a.out[1] + c - a.width[0], v);
}

// Tile and cuts of a product: the cheapest by a model of what was measured (us): a k tile of 64 takes a compute unit 2.2 with one large
// workgroup, 1.9 with two small ones and 1.2 with one (fp32, k tiles of 32: twice that; odd sizes
// another half), a workgroup 8 besides; the parts of a cut
// contraction are written and read at 4 TB/s and cost a launch.  What it decides: large tiles for many outputs, no round of workgroups
// that is almost empty, cuts for few outputs with a long contraction.
struct FfPlan { bool large; int tiles_m, tiles_n, cuts, cut_k; };
static FfPlan ff_plan(int dtype, bool gate, bool can_cut, int m, int n, int k) {
    FfPlan best = {};
    double best_cost = 1e30;
    const int bk = dtype == kF32 ? 32 : 64, k_tiles = k > 0 ? ceil_div(k, bk) : 1;
    for (int large = 0; large <= (dtype != kF32 ? 1 : 0); ++large) {
        const int side = large ? 256 : 128, tm = ceil_div(m, side), tn = ceil_div(n, gate ? side / 2 : side);
        const int64_t tiles = (int64_t)tm * tn;
        int last = 0;
        for (int want = 1; want <= (can_cut ? 64 : 1) && want <= k_tiles; ++want) {
            const int per = ceil_div(k_tiles, want), cuts = ceil_div(k_tiles, per);
            if (cuts == last) continue;
            last = cuts;
            const double blocks = (double)tiles * cuts, tile = (dtype == kF32 ? 2.0 : 1.0) * ((m | n | k) % 8 ? 1.5 : 1.0);
            double cost;
            if (large) cost = ceil(blocks / 256) * (2.2 * tile * per + 8);
            else cost = blocks <= 256 ? 1.2 * tile * per + 8 : ceil(blocks / 512) * (1.9 * tile * per + 8);
            if (cuts > 1) cost += 5 + (2.0 * cuts + 1) * m * n * 4e-6 / 4;
            if (cost < best_cost) {
                best_cost = cost;
                best = {large != 0, tm, tn, cuts, per * bk};
            }
        }
    }
    return best;
}
static int64_t ff_part_size(int dtype, int m, int n, int k) {
    const FfPlan p = ff_plan(dtype, false, true, m, n, k);
    return p.cuts > 1 ? (int64_t)p.cuts * m * n : 0;
}
template <int T, bool kAcrossA, bool kAcrossB, int kEpi>
static int ff_product(FfArgs<T> g, hipStream_t st, const char* what) {
    const FfPlan p = ff_plan(T, kEpi == kGate, kEpi == kPlain, g.m, g.n, g.k);
    g.tiles_m = p.tiles_m; g.tiles_n = p.tiles_n; g.cuts = p.cuts; g.cut_k = p.cut_k;
    const int64_t blocks = (int64_t)g.tiles_m * g.tiles_n * g.cuts;
    if (blocks == 0) return 0;
    EQ_CHECK_ARG(blocks < (1 << 23), EQUIGSPR_ENOTSUP, "%s: more workgroups than one launch takes", what);
    if constexpr (T != kF32) {
        if (p.large) ff_product_kernel<T, kAcrossA, kAcrossB, kEpi, true><<<(unsigned)blocks, 512, 0, st>>>(g);
    }
    if (!p.large) ff_product_kernel<T, kAcrossA, kAcrossB, kEpi, false><<<(unsigned)blocks, 256, 0, st>>>(g);
    EQ_CHECK_LAUNCH(what);
    if (g.cuts > 1) {
        const int64_t n = ceil_div((int64_t)g.m * g.n, 256);
        ff_sum_kernel<T><<<(unsigned)(n < 4096 ? n : 4096), 256, 0, st>>>(g);
        EQ_CHECK_LAUNCH(what);
    }
    return 0;
}

// both operands along the contraction, few rows: see ff_few_kernel.  Up to 32 rows, two blocks of 16: whole calls of 8 / 16 / 17 / 32 rows take
// 24 / 26 / 30 / 35 us against 41..43 by tiles (bf16, 2048 x 5632), 26 / 28 / 33 / 38 against 76 (fp32, 1024 x 4096), 15 against 20 (fp32, 32 x 128).
// Beyond, a third block's registers and the tiles' reuse of the weights count.
constexpr int kFewRows = 32;
template <int T, int kEpi>
static int ff_few(FfArgs<T> g, hipStream_t st, const char* what) {
    g.cut_k = ceil_div(ceil_div(g.k, kFewWaves), kFewStep) * kFewStep;
    const unsigned blocks = (unsigned)ceil_div(g.n, 16);
    if (g.m <= 16) ff_few_kernel<T, 1, kEpi><<<blocks, kFewWaves * 64, 0, st>>>(g);
    else ff_few_kernel<T, 2, kEpi><<<blocks, kFewWaves * 64, 0, st>>>(g);
    EQ_CHECK_LAUNCH(what);
    return 0;
}

template <int T>
static FfOperand<T> ff_operand(const void* p, int rows, int len) {
    using E = typename Num<T>::type;
    return {(const E*)p, (const E*)p, len, rows, rows, len};
}

template <int T>
static int ff_forward(const equigspr_gated_feed_forward* d, void* y, void* h, float* zu, float* work, hipStream_t st) {
    using E = typename Num<T>::type;
    FfArgs<T> g = {};
    g.act = d->activation;
    g.a = ff_operand<T>(d->x, d->rows, d->width);
    g.b = ff_operand<T>(d->w_gate, d->hidden, d->width);
    g.b.q = (const E*)d->w_up;
    g.m = d->rows; g.n = d->hidden; g.k = d->width;
    g.bias = (const E*)d->b_gate; g.bias2 = (const E*)d->b_up;
    g.c = (E*)h; g.zu = zu;
    const bool few = d->rows <= kFewRows;
    if (const int rc = few ? ff_few<T, kGate>(g, st, "gated_feed_forward (projections)") : ff_product<T, false, false, kGate>(g, st, "gated_feed_forward (projections)"))
        return rc;
    g.a = ff_operand<T>(h, d->rows, d->hidden);
    g.b = ff_operand<T>(d->w_down, d->out, d->hidden);
    g.n = d->out; g.k = d->hidden;
    g.bias = (const E*)d->b_down; g.bias2 = nullptr;
    g.c = (E*)y; g.zu = nullptr; g.part = work;
    return few ? ff_few<T, kPlain>(g, st, "gated_feed_forward (output)") : ff_product<T, false, false, kPlain>(g, st, "gated_feed_forward (output)");
}

template <int T>
static int ff_backward(const equigspr_gated_feed_forward* d, const void* gy, const float* zu, const void* h, void* dzu, float* work,
                       const equigspr_gated_feed_forward_grads* o, hipStream_t st) {
    using E = typename Num<T>::type;
    const int r = d->rows, w = d->width, hd = d->hidden, out = d->out;
    FfArgs<T> g = {};
    g.act = d->activation;
    const float* range = nullptr;
    if constexpr (T == kF16) {                // the first floats of the workspace
        ff_range_kernel<T><<<kFfRange, 1024, 0, st>>>((const E*)gy, (int64_t)r * out, work);
        EQ_CHECK_LAUNCH("gated_feed_forward_backward (range)");
        range = work;
        work += kFfRange;
    }
    g.range = range;
    // dh = dy Wd: rows of dy along the contraction (out), Wd [out, hidden] across it
    g.a = ff_operand<T>(gy, r, out);
    g.b = ff_operand<T>(d->w_down, out, hd);
    g.m = r; g.n = hd; g.k = out;
    g.zu = const_cast<float*>(zu); g.dzu = (E*)dzu;
    if (const int rc = ff_product<T, false, true, kGrad>(g, st, "gated_feed_forward_backward (hidden)")) return rc;
    g.zu = nullptr;
    g.dzu = nullptr;
    g.part = work;
    if (o->grad_x) {                          // [dz | du] [Wg ; Wu]
        g.a = ff_operand<T>(dzu, r, 2 * hd);
        g.b = ff_operand<T>(d->w_gate, 2 * hd, w);
        g.b.split = hd;
        g.b.q = (const E*)d->w_up;
        g.m = r; g.n = w; g.k = 2 * hd;
        g.c = (E*)o->grad_x;
        if (const int rc = ff_product<T, false, true, kPlain>(g, st, "gated_feed_forward_backward (input)")) return rc;
    }
    if (o->grad_w_gate_up) {                  // [dz | du]^T x
        g.a = ff_operand<T>(dzu, r, 2 * hd);
        g.b = ff_operand<T>(d->x, r, w);
        g.m = 2 * hd; g.n = w; g.k = r;
        g.c = (E*)o->grad_w_gate_up;
        if (const int rc = ff_product<T, true, true, kPlain>(g, st, "gated_feed_forward_backward (projections)")) return rc;
    }
    if (o->grad_w_down) {                     // dy^T h
        g.a = ff_operand<T>(gy, r, out);
        g.b = ff_operand<T>(h, r, hd);
        g.m = out; g.n = hd; g.k = r;
        g.range = nullptr;
        g.c = (E*)o->grad_w_down;
        if (const int rc = ff_product<T, true, true, kPlain>(g, st, "gated_feed_forward_backward (output)")) return rc;
    }
    if (o->grad_b_gate_up || o->grad_b_down) {
        FfColumns<T> c = {{(const E*)dzu, (const E*)gy}, {(E*)o->grad_b_gate_up, (E*)o->grad_b_down}, {o->grad_b_gate_up ? 2 * hd : 0, o->grad_b_down ? out : 0},
                          r, ceil_div(r, kFfRun), range};
        ff_columns_kernel<T><<<dim3(ceil_div(c.width[0], 64) + ceil_div(c.width[1], 64), c.runs), 256, 0, st>>>(c, work);
        EQ_CHECK_LAUNCH("gated_feed_forward_backward (biases)");
        ff_columns_sum_kernel<T><<<ceil_div(c.width[0] + c.width[1], 64), 256, 0, st>>>(c, work);
        EQ_CHECK_LAUNCH("gated_feed_forward_backward (biases' runs)");
    }
    return 0;
}

static int ff_check(const equigspr_gated_feed_forward* d) {
    EQ_CHECK_ARG(d, EQUIGSPR_EINVAL, "gated_feed_forward: null description");
    EQ_CHECK_ARG(d->dtype == EQUIGSPR_F32 || d->dtype == EQUIGSPR_BF16 || d->dtype == EQUIGSPR_F16, EQUIGSPR_EINVAL, "gated_feed_forward: unknown dtype %d", d->dtype);
    EQ_CHECK_ARG(d->activation == kSilu || d->activation == kGelu || d->activation == kRelu, EQUIGSPR_EINVAL, "gated_feed_forward: unknown activation %d", d->activation);
    EQ_CHECK_ARG(d->rows >= 0 && d->width >= 1 && d->hidden >= 1 && d->out >= 1, EQUIGSPR_EINVAL, "gated_feed_forward: bad sizes");
    EQ_CHECK_ARG(d->rows <= 65535 * kFfRun && d->width < (1 << 20) && d->hidden < (1 << 20) && d->out < (1 << 20), EQUIGSPR_ENOTSUP, "gated_feed_forward: sizes beyond the kernels' range");
    EQ_CHECK_ARG(d->w_gate && d->w_up && d->w_down && (d->x || !d->rows), EQUIGSPR_EINVAL, "gated_feed_forward: null tensor");
    return 0;
}

}  // namespace eq

extern "C" int64_t equigspr_gated_feed_forward_work_size(const equigspr_gated_feed_forward* d) {
    if (eq::ff_check(d) != 0) return -1;
    return d->rows <= eq::kFewRows ? 0 : eq::ff_part_size(d->dtype, d->rows, d->out, d->hidden);
}

extern "C" int equigspr_gated_feed_forward_forward(const equigspr_gated_feed_forward* d, void* y, void* h, float* zu, float* work, void* stream) {
    if (const int rc = eq::ff_check(d)) return rc;
    if (d->rows == 0) return 0;
    EQ_CHECK_ARG(y && h && (work || equigspr_gated_feed_forward_work_size(d) == 0), EQUIGSPR_EINVAL, "gated_feed_forward_forward: null output or work");
    hipStream_t st = (hipStream_t)stream;
    switch (d->dtype) {
        case EQUIGSPR_F32: return eq::ff_forward<eq::kF32>(d, y, h, zu, work, st);
        case EQUIGSPR_BF16: return eq::ff_forward<eq::kBF16>(d, y, h, zu, work, st);
        default: return eq::ff_forward<eq::kF16>(d, y, h, zu, work, st);
    }
}

extern "C" int64_t equigspr_gated_feed_forward_backward_work_size(const equigspr_gated_feed_forward* d) {
    if (eq::ff_check(d) != 0) return -1;
    int64_t n = eq::ff_part_size(d->dtype, d->rows, d->width, 2 * d->hidden);
    const int64_t up = eq::ff_part_size(d->dtype, 2 * d->hidden, d->width, d->rows), down = eq::ff_part_size(d->dtype, d->out, d->hidden, d->rows);
    const int64_t sums = (int64_t)eq::ceil_div(d->rows, eq::kFfRun) * (2 * d->hidden + d->out);
    n = up > n ? up : n;
    n = down > n ? down : n;
    return (sums > n ? sums : n) + (d->dtype == EQUIGSPR_F16 ? eq::kFfRange : 0);
}

extern "C" int equigspr_gated_feed_forward_backward(const equigspr_gated_feed_forward* d, const void* grad_y, const float* zu, const void* h, void* dzu, float* work,
                                                    const equigspr_gated_feed_forward_grads* grads, void* stream) {
    if (const int rc = eq::ff_check(d)) return rc;
    if (d->rows == 0) return 0;
    EQ_CHECK_ARG(grad_y && zu && h && dzu && work && grads, EQUIGSPR_EINVAL, "gated_feed_forward_backward: null tensor");
    hipStream_t st = (hipStream_t)stream;
    switch (d->dtype) {
        case EQUIGSPR_F32: return eq::ff_backward<eq::kF32>(d, grad_y, zu, h, dzu, work, grads, st);
        case EQUIGSPR_BF16: return eq::ff_backward<eq::kBF16>(d, grad_y, zu, h, dzu, work, grads, st);
        default: return eq::ff_backward<eq::kF16>(d, grad_y, zu, h, dzu, work, grads, st);
    }
}
