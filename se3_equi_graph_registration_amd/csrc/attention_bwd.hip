// Attention between the points of clouds, backward.  The probabilities are recomputed from the forward's log-sums L:
//   P = exp2(c S - L),  delta = rowsum(dO * O),  dV = P^T dO,  dP = dO V^T,  dS = P * (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q.
// Two kernels, seven products: attn_dq_kernel owns 32 packed rows per wave and walks the keys (it also computes delta, once);
// attn_dkv_kernel owns 32 keys per wave and walks the packed rows -- all query heads of the group, so the gradients of shared keys need
// no atomics and do not depend on timing.  In each, the score tile is formed with the owned index in the lane, which makes P and dS the
// B operands of the products that follow as they stand (see attention.hip); the other operand is the staged tile read transposed.
// P and dS are rounded to the inputs' 16-bit type for those products (heads of up to 16 dims take a second plane with what that
// drops), everything else is fp32; the forward leaves what the output's rounding dropped in a second plane for delta, whose error every
// dS of the row would share.
// Bound: as the forward (matrix pipe busy 0.31 / 0.36 at heads of 64 in the two kernels, 0.47 / 0.37 at 128), and the registers -- the
// accumulators of wide heads leave two waves per SIMD, and the keys' kernel at 97..128 dims spills (bf16 43, fp16 28 registers, 80 bytes).
// Measured, bf16: 8 x 2048^2 x 8 heads of 64 285 us (600 TFLOP/s of the five products that the mathematics needs), 8192^2 x 16 / 4 heads of 128
// 2.0 ms (690), causal 1.15 ms.
// fp16: dS is about 1/keys of the output gradient and would sink below fp16's range, so it is held as 2^E dS, with E from the largest
// |dO| and |V| of the sample and key head such that the bound |dS| <= 2 dim max|dO| max|V| stays in range; undone in fp32 at the end.
// (One E for a whole batch would let one sample's or head's large gradients push the others' into fp16's smallest steps.)
#include "attention_device.h"

namespace eq {

template <int T>
struct AttnBwd {
    AttnShape s;
    AttnTensor<T> q, k, v, o, g;              // g: gradient of the output
    const typename Num<T>::type* o_low;       // 16-bit types: what the output's rounding dropped, or null
    const float* lse;
    float* delta;                             // [batch, kv_heads, nq * group]
    float* amax;                              // fp16: [batch * kv_heads][amax_parts][2], largest |dO| and |V|
    int amax_parts;                           // <= 64
    typename Num<T>::type *gq, *gk, *gv;      // contiguous, each may be null
    int row_tiles, key_tiles;
    int key_splits, split_keys;               // attn_dq_kernel: parts of the key axis
    int row_splits;                           // attn_dkv_kernel: parts of the row axis
    float *part_q, *part_k, *part_v;          // [splits][the gradient's elements] when an axis is split
};

// rows of a staged tile: 64, or 32 where three planes or a wide head would take the registers of a second wave per SIMD
template <int T, int W> constexpr int attn_bwd_tile() { return W == 128 || (T == kF32 && W == 64) ? 32 : 64; }

// fp16: largest |dO| over the rows with a visible key and |V| over the visible keys of a sample and key head, one pair per workgroup
template <int T>
__global__ __launch_bounds__(256) void attn_amax_kernel(AttnBwd<T> a) {
    const AttnShape& s = a.s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int bh = blockIdx.x / a.amax_parts, at = blockIdx.x - bh * a.amax_parts, b = bh / s.kv_heads, hk = bh - b * s.kv_heads;
    float mg = 0.f, mv = 0.f;
    // a thread per chunk of eight values: as many whole rows at a time as fit the workgroup
    const int chunks = (s.dim + 7) / 8, per = 256 / chunks, r0 = threadIdx.x / chunks, c = threadIdx.x - r0 * chunks;
    auto most = [&](float& m, const typename Num<T>::type* row) {
        const Raw8<T> r = load8<T>(row, 8 * c, s.dim);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(raw_float<T>(r, i)));
    };
    const int rows = attn_len(s.q_lens, b, s.nq) * s.group, keys = attn_len(s.kv_lens, b, s.nk);
    if (r0 < per) {
        for (int r = at * per + r0; r < rows; r += a.amax_parts * per)
            if (a.lse[(int64_t)bh * s.nq * s.group + r] != INFINITY) most(mg, packed_row(a.g, s, b, hk, r));
        for (int j = at * per + r0; j < keys; j += a.amax_parts * per)
            if (!s.key_mask || s.key_mask[b * s.mask_stride + j]) most(mv, key_row(a.v, b, hk, j));
    }
    __shared__ float part[2][4];
    for (int o = 32; o; o >>= 1) { mg = fmaxf(mg, __shfl_xor(mg, o)); mv = fmaxf(mv, __shfl_xor(mv, o)); }
    if (lane == 0) { part[0][wave] = mg; part[1][wave] = mv; }
    __syncthreads();
    if (threadIdx.x < 2)
        a.amax[2 * blockIdx.x + threadIdx.x] = fmaxf(fmaxf(part[threadIdx.x][0], part[threadIdx.x][1]), fmaxf(part[threadIdx.x][2], part[threadIdx.x][3]));
}
// enough workgroups for the card when there are few heads; a wave joins a head's parts with one load
static int attn_amax_parts(int64_t heads) { return heads >= 1024 ? 1 : heads <= 16 ? 64 : (int)(1024 / heads); }

// the power of two dS is held with: 1 except in fp16
template <int T>
__device__ __forceinline__ float attn_grad_scale(const AttnBwd<T>& a, int bh) {
    if constexpr (T != kF16) return 1.f;
    const int lane = threadIdx.x & 63;
    float mg = 0.f, mv = 0.f;
    if (lane < a.amax_parts) {
        const float* p = a.amax + 2 * ((int64_t)bh * a.amax_parts + lane);
        mg = p[0];
        mv = p[1];
    }
    for (int o = 32; o; o >>= 1) { mg = fmaxf(mg, __shfl_xor(mg, o)); mv = fmaxf(mv, __shfl_xor(mv, o)); }
    const float bound = 2.f * a.s.dim * mg * mv;
    if (!(bound > 0.f) || bound > 3e38f) return 1.f;
    const int e = (int)floorf(log2f(60000.f) - log2f(bound));
    return ldexpf(1.f, e < -60 ? -60 : (e > 60 ? 60 : e));
}

constexpr int kBwdWaves = 4;                  // waves of a workgroup: each owns 32 rows (keys), all share the staged tiles

template <int T, int W, int KS>
__global__ __launch_bounds__(kBwdWaves * 64, T == kF32 ? 1 : 2) void attn_dq_kernel(AttnBwd<T> a) {
    constexpr int KT = attn_bwd_tile<T, W>(), NT = kBwdWaves * 64, ROWS = kBwdWaves * 32, NP = Num<T>::planes;
    constexpr int DB = (KS + 1) / 2, KB = KT / 32;
    __shared__ __attribute__((aligned(16))) short tile_k[NP * Tile<W>::size(KT)];
    __shared__ __attribute__((aligned(16))) short tile_v[NP * Tile<W>::size(KT)];
    __shared__ __attribute__((aligned(16))) float hidden[KT];
    const AttnShape& s = a.s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const AttnUnit un = attn_unit(s.batch * s.kv_heads, a.row_tiles * a.key_splits);
    const int rt = a.row_tiles - 1 - un.unit / a.key_splits, split = un.unit % a.key_splits, bh = un.bh, b = bh / s.kv_heads, hk = bh - b * s.kv_heads;
    const int ql = attn_len(s.q_lens, b, s.nq), kl = attn_len(s.kv_lens, b, s.nk);
    const int rows = s.nq * s.group, rows_valid = ql * s.group, row0 = rt * ROWS;
    const int row = row0 + wave * 32 + (lane & 31);
    const bool ok_row = row < rows_valid;
    const int k_begin = split * a.split_keys;
    int k_end = min(kl, k_begin + a.split_keys);
    const int last_row = min(row0 + ROWS, rows_valid) - 1;
    if (s.causal && last_row >= 0) k_end = min(k_end, row_point(s, last_row) + kl - ql + 1);
    if (row0 >= rows_valid || !a.gq) k_end = 0;
    const int limit = s.causal ? row_point(s, row) + kl - ql : 0x7fffffff;
    const uint8_t* mask = s.key_mask ? s.key_mask + b * s.mask_stride : nullptr;
    const int64_t at = (int64_t)bh * rows + row;

    // A row without a visible key takes no gradient, whatever it and its output gradient hold: both become zeros (after their loads, which
    // need not wait for the log-sum).
    const float lse = ok_row ? a.lse[at] : INFINITY;
    Op8<T> q[KS], g[KS];
    float delta = 0.f;
    {
        const typename Num<T>::type* pq = ok_row ? packed_row(a.q, s, b, hk, row) : nullptr;
        const typename Num<T>::type* pg = ok_row ? packed_row(a.g, s, b, hk, row) : nullptr;
        const typename Num<T>::type* po = ok_row ? packed_row(a.o, s, b, hk, row) : nullptr;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int c = ks * 16 + half * 8;
            Raw8<T> rq = ok_row ? load8<T>(pq, c, s.dim) : raw_zero<T>(), rg = ok_row ? load8<T>(pg, c, s.dim) : raw_zero<T>();
            const Raw8<T> ro = ok_row ? load8<T>(po, c, s.dim) : raw_zero<T>();
            if (lse == INFINITY) rq = rg = raw_zero<T>();
            q[ks] = planes_of<T>(rq);
#pragma unroll
            for (int i = 0; i < 8; ++i) delta = fmaf(raw_float<T>(rg, i), raw_float<T>(ro, i), delta);
            if (T != kF32 && a.o_low && ok_row) {
                const Raw8<T> rl = load8<T>(a.o_low + (po - a.o.p), c, s.dim);
#pragma unroll
                for (int i = 0; i < 8; ++i) delta = fmaf(raw_float<T>(rg, i), raw_float<T>(rl, i), delta);
            }
            g[ks] = planes_of<T>(rg);
        }
    }
    delta += __shfl_xor(delta, 32);
    if (row < rows && half == 0 && split == 0) a.delta[at] = delta;
    if (!a.gq) return;
    const float factor = attn_grad_scale<T>(a, bh);
    pf32x16 acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;

    Stager<T, W, KT, NT> sk, sv;
    sk.init([&](int j) { return j * (int)a.k.sn; });
    sv.init([&](int j) { return j * (int)a.v.sn; });
    bool vis = false;
    const bool even = !mask && s.dim % 8 == 0;
    auto load_tile = [&](int k0) {
        if (even && k0 + KT <= k_end) {
            sk.load_whole(key_row(a.k, b, hk, k0), s.dim);
            sv.load_whole(key_row(a.v, b, hk, k0), s.dim);
            vis = true;
            return;
        }
        auto ok = [&](int j) { return k0 + j < k_end && (!mask || mask[k0 + j]); };
        sk.load([&](int j) { return ok(j) ? key_row(a.k, b, hk, k0 + j) : nullptr; }, s.dim);
        sv.load([&](int j) { return ok(j) ? key_row(a.v, b, hk, k0 + j) : nullptr; }, s.dim);
        if (threadIdx.x < KT) vis = ok(threadIdx.x);
    };
    if (k_begin < k_end) load_tile(k_begin);
    for (int k0 = k_begin; k0 < k_end; k0 += KT) {
        __syncthreads();
        sk.store(tile_k);
        sv.store(tile_v);
        if (threadIdx.x < KT) hidden[threadIdx.x] = vis ? 0.f : 1.f;
        __syncthreads();
        if (k0 + KT < k_end) load_tile(k0 + KT);
        const bool edge = mask || k0 + KT > k_end || (s.causal && k0 + KT > row_point(s, row0 + wave * 32) + kl - ql + 1);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            pf32x16 sc, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[r] = dp[r] = 0.f;
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                mma<T>(sc, tile_rows<T, W, KT>(tile_k, kb * 32, ks, lane), q[ks]);
                mma<T>(dp, tile_rows<T, W, KT>(tile_v, kb * 32, ks, lane), g[ks]);
            }
            __builtin_amdgcn_s_setprio(0);
            if (edge) {
                asm volatile("");                         // a branch: as selects this would be a third of the tile's arithmetic
#pragma unroll
                for (int gq = 0; gq < 4; ++gq) {
                    const int j = kb * 32 + 8 * gq + 4 * half;
                    const pf32x4 h = *reinterpret_cast<const pf32x4*>(hidden + j);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (h[i] != 0.f || k0 + j + i > limit) sc[4 * gq + i] = -INFINITY;
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    x[j] = exp2_fast(fmaf(sc[8 * t + j], s.scale_log2, -lse)) * (dp[8 * t + j] - delta) * factor;
                const Op8<T> ds = pack8<T>(x);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const Op8<T> kt = tile_cols<T, W, KT>(tile_k, kb * 32 + 16 * t, d * 32, lane);
                    if constexpr (attn_two_planes<T, KS>()) mma<T>(acc[d], kt, pack8_rest<T>(x));
                    mma<T>(acc[d], kt, ds);
                }
            }
        }
    }
    if (row >= rows) return;
    const float back = s.scale / factor;
    const int i0 = row_point(s, row);
    const int64_t o = (((int64_t)b * s.nq + i0) * s.heads + hk * s.group + row - i0 * s.group) * s.dim;
    float* part = a.key_splits > 1 ? a.part_q + split * (int64_t)s.batch * s.nq * s.heads * s.dim : nullptr;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int gq = 0; gq < 4; ++gq) {
            const int c = d * 32 + 8 * gq + 4 * half;
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = acc[d][4 * gq + i] * back;
            if (part) store4<kF32>(part + o + c, x, s.dim - c);
            else store4<T>(a.gq + o + c, x, s.dim - c);
        }
}

// kDeadRows: rows without a visible key may lie among those that reach this tile's keys (a mask hides what causal leaves) and are left out.  A
// form of its own: the test for it in the others' loads cost heads of 128 another 60 spilled registers (8192^2 causal: 1449 us instead of 1425).
template <int T, int W, int KS, bool kDeadRows>
__global__ __launch_bounds__(kBwdWaves * 64, T == kF32 ? 1 : 2) void attn_dkv_kernel(AttnBwd<T> a) {
    constexpr int RT = attn_bwd_tile<T, W>(), NT = kBwdWaves * 64, KEYS = kBwdWaves * 32, NP = Num<T>::planes;
    constexpr int DB = (KS + 1) / 2, RB = RT / 32;
    constexpr float kShift = T == kF16 ? 10.f : 0.f;
    __shared__ __attribute__((aligned(16))) short tile_q[NP * Tile<W>::size(RT)];
    __shared__ __attribute__((aligned(16))) short tile_g[NP * Tile<W>::size(RT)];
    __shared__ __attribute__((aligned(16))) float row_lse[RT];
    __shared__ __attribute__((aligned(16))) float row_delta[RT];
    __shared__ __attribute__((aligned(16))) int row_limit[RT];
    // wide 16-bit heads: V waits in LDS, its registers make room for a second wave per SIMD
    constexpr bool kKeepV = !(W == 128 && NP == 1);
    __shared__ __attribute__((aligned(16))) short own_v[kKeepV ? 8 : Tile<W>::size(KEYS)];
    const AttnShape& s = a.s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const AttnUnit un = attn_unit(s.batch * s.kv_heads, a.key_tiles * a.row_splits);
    const int kt = un.unit / a.row_splits, split = un.unit % a.row_splits, bh = un.bh, b = bh / s.kv_heads, hk = bh - b * s.kv_heads;
    const int ql = attn_len(s.q_lens, b, s.nq), kl = attn_len(s.kv_lens, b, s.nk);
    const int rows = s.nq * s.group, rows_valid = ql * s.group, key0 = kt * KEYS;
    const int key = key0 + wave * 32 + (lane & 31);
    const bool ok_key = key < kl && (!s.key_mask || s.key_mask[b * s.mask_stride + key]);
    // the rows from the first point that sees this tile's first key, cut into equal parts
    const int r_first = s.causal ? max(0, key0 - kl + ql) * s.group : 0, r_count = key0 < kl ? max(0, rows_valid - r_first) : 0;
    const int r_part = ((r_count + a.row_splits - 1) / a.row_splits + RT - 1) / RT * RT;
    const int r_begin = r_first + split * r_part, r_end = min(r_first + r_count, r_begin + r_part);

    Op8<T> k[KS], v[kKeepV ? KS : 1];                      // keys that are not visible: zeros; their lanes' results are replaced at the end
    {
        const typename Num<T>::type* pk = ok_key ? key_row(a.k, b, hk, key) : nullptr;
        const typename Num<T>::type* pv = ok_key ? key_row(a.v, b, hk, key) : nullptr;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int c = ks * 16 + half * 8;
            k[ks] = planes_of<T>(ok_key ? load8<T>(pk, c, s.dim) : raw_zero<T>());
            const Op8<T> o = planes_of<T>(ok_key ? load8<T>(pv, c, s.dim) : raw_zero<T>());
            if constexpr (kKeepV) v[ks] = o;
            else *reinterpret_cast<s16x8*>(own_v + Tile<W>::at(wave * 32 + (lane & 31), 2 * ks + half)) = o.p[0];
        }
    }
    const float factor = attn_grad_scale<T>(a, bh), fs = factor * exp2_fast(-kShift);
    pf32x16 acc_k[DB], acc_v[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc_k[d][r] = acc_v[d][r] = 0.f;

    Stager<T, W, RT, NT> sq, sg;
    sq.init([&](int r) { const int i = row_point(s, r); return i * (int)a.q.sn + (r - i * s.group) * (int)a.q.sh; });
    sg.init([&](int r) { const int i = row_point(s, r); return i * (int)a.g.sn + (r - i * s.group) * (int)a.g.sh; });
    const bool even = !kDeadRows && RT % s.group == 0 && s.dim % 8 == 0;       // tiles then begin with the first head of a group
    float my_lse = INFINITY, my_delta = 0.f;
    int my_limit = -1;
    auto load_tile = [&](int r0) {
        if (even && r0 + RT <= r_end) {
            sq.load_whole(packed_row(a.q, s, b, hk, r0), s.dim);
            sg.load_whole(packed_row(a.g, s, b, hk, r0), s.dim);
        } else {
            auto ok = [&](int r) { return r < r_end && (!kDeadRows || a.lse[(int64_t)bh * rows + r] != INFINITY); };
            sq.load([&](int r) { return ok(r0 + r) ? packed_row(a.q, s, b, hk, r0 + r) : nullptr; }, s.dim);
            sg.load([&](int r) { return ok(r0 + r) ? packed_row(a.g, s, b, hk, r0 + r) : nullptr; }, s.dim);
        }
        if (threadIdx.x < RT) {
            const int r = r0 + threadIdx.x;
            const int64_t at = (int64_t)bh * rows + r;
            my_lse = r < r_end ? a.lse[at] : INFINITY;
            my_delta = r < r_end ? a.delta[at] : 0.f;
            my_limit = row_point(s, r) + kl - ql;
        }
    };
    if (r_begin < r_end) load_tile(r_begin);
    for (int r0 = r_begin; r0 < r_end; r0 += RT) {
        __syncthreads();
        sq.store(tile_q);
        sg.store(tile_g);
        if (threadIdx.x < RT) { row_lse[threadIdx.x] = kShift - my_lse; row_delta[threadIdx.x] = my_delta; row_limit[threadIdx.x] = my_limit; }
        __syncthreads();
        if (r0 + RT < r_end) load_tile(r0 + RT);
        const bool edge = s.causal && key0 + wave * 32 + 31 > row_point(s, r0) + kl - ql;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            pf32x16 sc, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[r] = dp[r] = 0.f;
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                mma<T>(sc, tile_rows<T, W, RT>(tile_q, rb * 32, ks, lane), k[ks]);
                Op8<T> ov;
                if constexpr (kKeepV) ov = v[ks];
                else ov.p[0] = Tile<W>::row8(own_v, wave * 32 + (lane & 31), 2 * ks + half);      // written by this wave
                mma<T>(dp, tile_rows<T, W, RT>(tile_g, rb * 32, ks, lane), ov);
            }
#pragma unroll
            for (int gr = 0; gr < 4; ++gr) {
                const int r = rb * 32 + 8 * gr + 4 * half;
                const pf32x4 sub = *reinterpret_cast<const pf32x4*>(row_lse + r), del = *reinterpret_cast<const pf32x4*>(row_delta + r);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = exp2_fast(fmaf(sc[4 * gr + i], s.scale_log2, sub[i]));
                    sc[4 * gr + i] = p;
                    dp[4 * gr + i] = p * (dp[4 * gr + i] - del[i]) * fs;
                }
            }
            __builtin_amdgcn_s_setprio(0);
            if (edge) {
                asm volatile("");                         // a branch, see above
#pragma unroll
                for (int gr = 0; gr < 4; ++gr)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (key > row_limit[rb * 32 + 8 * gr + 4 * half + i]) sc[4 * gr + i] = dp[4 * gr + i] = 0.f;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float x[8], y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) { x[j] = sc[8 * t + j]; y[j] = dp[8 * t + j]; }
                const Op8<T> p = pack8<T>(x), ds = pack8<T>(y);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const Op8<T> gt = tile_cols<T, W, RT>(tile_g, rb * 32 + 16 * t, d * 32, lane), qt = tile_cols<T, W, RT>(tile_q, rb * 32 + 16 * t, d * 32, lane);
                    if constexpr (attn_two_planes<T, KS>()) {
                        mma<T>(acc_v[d], gt, pack8_rest<T>(x));
                        mma<T>(acc_k[d], qt, pack8_rest<T>(y));
                    }
                    mma<T>(acc_v[d], gt, p);
                    mma<T>(acc_k[d], qt, ds);
                }
            }
        }
    }
    if (key >= s.nk) return;
    const float back_k = s.scale / factor, back_v = exp2_fast(-kShift);
    const int64_t o = (((int64_t)b * s.nk + key) * s.kv_heads + hk) * s.dim;
    const int64_t part = a.row_splits > 1 ? split * (int64_t)s.batch * s.nk * s.kv_heads * s.dim : -1;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int gr = 0; gr < 4; ++gr) {
            const int c = d * 32 + 8 * gr + 4 * half;
            float x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = ok_key ? acc_k[d][4 * gr + i] * back_k : 0.f;
                y[i] = ok_key ? acc_v[d][4 * gr + i] * back_v : 0.f;
            }
            if (part >= 0) {
                if (a.gk) store4<kF32>(a.part_k + part + o + c, x, s.dim - c);
                if (a.gv) store4<kF32>(a.part_v + part + o + c, y, s.dim - c);
            } else {
                if (a.gk) store4<T>(a.gk + o + c, x, s.dim - c);
                if (a.gv) store4<T>(a.gv + o + c, y, s.dim - c);
            }
        }
}

// a gradient as the sum of its parts, in order; the two gradients of keys and values in one launch
template <int T>
__global__ __launch_bounds__(256) void attn_sum_kernel(const float* part0, const float* part1, int splits, int64_t n, typename Num<T>::type* out0,
                                                       typename Num<T>::type* out1) {
    const float* part = blockIdx.y ? part1 : part0;
    typename Num<T>::type* out = blockIdx.y ? out1 : out0;
    if (!out) return;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int p = 0; p < splits; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n) v[e] += part[p * n + i + e];
        store4<T>(out + i, v, (int)(n - i < 4 ? n - i : 4));
    }
}

// Parts: the owned axis alone gives too few workgroups when it is short, and a causal mask leaves the first keys with all the work, so the
// other axis is cut until there are two workgroups per compute unit (causal: four), one part for every 256 of
// its length at most (257 are cut into 192 and 65; with whole parts of 256 alone, fp32 heads of 8 at 2 x 300^2 took 51 us instead of 44, heads of
// 32 at 2 x 700^2 73 instead of 64).
static int attn_bwd_splits(int64_t tiles, int64_t length, int64_t want) {
    if (tiles == 0 || tiles >= want) return 1;
    const int64_t most = (length + 255) / 256, s = want / tiles;
    return (int)(s < most ? (s > 1 ? s : 1) : (most > 1 ? most : 1));
}

struct AttnBwdPlan { int row_tiles, key_tiles, key_splits, split_keys, row_splits; int amax_parts; int64_t amax, delta, parts_q, parts_k; };
static AttnBwdPlan attn_bwd_plan(const AttnShape& s) {
    constexpr int kOwned = kBwdWaves * 32;
    AttnBwdPlan p;
    const int64_t heads = (int64_t)s.batch * s.kv_heads, rows = (int64_t)s.nq * s.group;
    p.row_tiles = ceil_div(rows, kOwned);
    p.key_tiles = ceil_div(s.nk, kOwned);
    p.key_splits = attn_bwd_splits(p.row_tiles * heads, s.nk, 512);
    p.split_keys = ceil_div(ceil_div(s.nk, p.key_splits), 64) * 64;
    p.key_splits = s.nk ? ceil_div(s.nk, p.split_keys) : 1;
    p.row_splits = attn_bwd_splits(p.key_tiles * heads, rows, s.causal ? 1024 : 512);
    p.amax_parts = attn_amax_parts(heads);
    p.amax = (2 * heads * p.amax_parts + 3) / 4 * 4;
    p.delta = (heads * rows + 3) / 4 * 4;
    p.parts_q = p.key_splits > 1 ? p.key_splits * heads * rows * s.dim : 0;
    p.parts_k = p.row_splits > 1 ? p.row_splits * heads * s.nk * s.dim : 0;
    return p;
}

template <int T, int W, int KS>
static int attn_bwd_launch(const AttnBwd<T>& a, hipStream_t st) {
    const AttnShape& s = a.s;
    const int64_t heads = (int64_t)s.batch * s.kv_heads;
    const int64_t bq = (int64_t)a.row_tiles * a.key_splits * heads, bk = (int64_t)a.key_tiles * a.row_splits * heads;
    EQ_CHECK_ARG(bq < (1 << 24) && bk < (1 << 24), EQUIGSPR_ENOTSUP, "attention_backward: more workgroups than one launch takes");
    if constexpr (T == kF16) {
        attn_amax_kernel<T><<<(unsigned)(heads * a.amax_parts), 256, 0, st>>>(a);
        EQ_CHECK_LAUNCH("attention_backward (range)");
    }
    if (bq) {
        attn_dq_kernel<T, W, KS><<<(unsigned)bq, kBwdWaves * 64, 0, st>>>(a);
        EQ_CHECK_LAUNCH("attention_backward (rows)");
        if (a.key_splits > 1 && a.gq) {
            const int64_t n = heads * s.nq * s.group * s.dim, blocks = ceil_div(n, 1024);
            attn_sum_kernel<T><<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, st>>>(a.part_q, nullptr, a.key_splits, n, a.gq, nullptr);
            EQ_CHECK_LAUNCH("attention_backward (rows' parts)");
        }
    }
    if (bk && (a.gk || a.gv)) {
        if (s.key_mask && s.causal) attn_dkv_kernel<T, W, KS, true><<<(unsigned)bk, kBwdWaves * 64, 0, st>>>(a);
        else attn_dkv_kernel<T, W, KS, false><<<(unsigned)bk, kBwdWaves * 64, 0, st>>>(a);
        EQ_CHECK_LAUNCH("attention_backward (keys)");
        if (a.row_splits > 1) {
            const int64_t n = heads * s.nk * s.dim, blocks = ceil_div(n, 1024);
            attn_sum_kernel<T><<<dim3((unsigned)(blocks < 4096 ? blocks : 4096), 2), 256, 0, st>>>(a.part_k, a.part_v, a.row_splits, n, a.gk, a.gv);
            EQ_CHECK_LAUNCH("attention_backward (keys' parts)");
        }
    }
    return 0;
}

template <int T>
static int attn_bwd(const equigspr_attention* d, const AttnShape& s, const void* out, const void* out_low, const float* lse,
                    const equigspr_attention_tensor* grad_out, float* work, void* gq, void* gk, void* gv, hipStream_t st) {
    using E = typename Num<T>::type;
    AttnBwd<T> a;
    a.s = s;
    a.q = attn_tensor<T>(d->q, s.dim);
    a.k = attn_tensor<T>(d->k, s.dim);
    a.v = attn_tensor<T>(d->v, s.dim);
    a.g = attn_tensor<T>(*grad_out, s.dim);
    const equigspr_attention_tensor o = {const_cast<void*>(out), (int64_t)s.nq * s.heads * s.dim, (int64_t)s.heads * s.dim, s.dim};
    a.o = attn_tensor<T>(o, s.dim);
    a.o_low = (const E*)out_low;
    a.lse = lse;
    a.amax = work;
    const AttnBwdPlan p = attn_bwd_plan(s);
    a.amax_parts = p.amax_parts;
    a.delta = work + p.amax;
    a.part_q = a.part_k = a.delta + p.delta;  // the rows' parts are summed before the keys' parts are written
    a.part_v = a.part_k + p.parts_k;
    a.row_tiles = p.row_tiles; a.key_tiles = p.key_tiles; a.key_splits = p.key_splits; a.split_keys = p.split_keys; a.row_splits = p.row_splits;
    a.gq = (E*)gq; a.gk = (E*)gk; a.gv = (E*)gv;
    return EQ_ATTN_BY_DIM(attn_bwd_launch, s.dim, a, st);
}

}  // namespace eq

extern "C" int64_t equigspr_attention_backward_work_size(const equigspr_attention* d) {
    eq::AttnShape s;
    if (eq::attn_shape(d, &s) != 0) return -1;
    const eq::AttnBwdPlan p = eq::attn_bwd_plan(s);
    return p.amax + p.delta + (p.parts_q > 2 * p.parts_k ? p.parts_q : 2 * p.parts_k);
}

extern "C" int equigspr_attention_backward(const equigspr_attention* d, const void* out, const void* out_low, const float* lse,
                                           const equigspr_attention_tensor* grad_out, float* work, void* grad_q, void* grad_k, void* grad_v, void* stream) {
    eq::AttnShape s;
    if (const int rc = eq::attn_shape(d, &s)) return rc;
    EQ_CHECK_ARG(grad_out && work, EQUIGSPR_EINVAL, "attention_backward: grad_out or work is null");
    EQ_CHECK_ARG(eq::attn_near(*grad_out, d->dtype == EQUIGSPR_F32 ? 4 : 2), EQUIGSPR_ENOTSUP, "attention_backward: strides of grad_out out of range");
    EQ_CHECK_ARG(!s.batch || !s.nq || (out && lse && grad_out->data), EQUIGSPR_EINVAL, "attention_backward: out, lse or grad_out is null");
    if (s.batch == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    switch (d->dtype) {
        case EQUIGSPR_F32: return eq::attn_bwd<eq::kF32>(d, s, out, out_low, lse, grad_out, work, grad_q, grad_k, grad_v, st);
        case EQUIGSPR_BF16: return eq::attn_bwd<eq::kBF16>(d, s, out, out_low, lse, grad_out, work, grad_q, grad_k, grad_v, st);
        default: return eq::attn_bwd<eq::kF16>(d, s, out, out_low, lse, grad_out, work, grad_q, grad_k, grad_v, st);
    }
}
