// Attention between the points of clouds, forward (cloud_attention):  S = c Q K^T,  P = softmax over the allowed keys,  O = P V.
//
// One pass over the keys with the running maximum and sum of the softmax; S and P never leave the registers.  A wave owns 32 packed
// rows (attention_device.h): the products are formed transposed, S^T = K Q^T (C tile: lane = row, registers = keys), so the softmax of
// a row is a loop over one lane's registers plus one exchange with lane ^ 32, and P^T is the B operand of O^T = V^T P^T as it stands
// (tile_cols reads V in the matching key order).  Statistics, P and O are fp32; P is rounded to the inputs' 16-bit type for the second
// product (at most 2^-8 / 2^-11 of each probability, averaged over the keys; heads of up to 16 dims take a second plane with what that
// drops, fp32 keeps all three).
// Few rows against many keys: the key axis is split over workgroups, each writes its normalised part and its log-sum, and
// attn_join_kernel joins them in split order (no atomics: results do not depend on timing).
// Bound: how little softmax and products overlap.  By counters, heads of 64: the vector ALU is busy 0.56 of the time, the matrix pipe 0.31 (a
// 64-key tile costs a wave 160 instructions of softmax, 32 of them exponentials, beside 16 products), heads of 128: 0.44 and 0.44; a wave does
// one after the other, and what the other waves of its SIMD fill in leaves the rest idle.  Few rows: HBM.  Measured, bf16: 8 x 2048^2 x 8 heads
// of 64 104..110 us (625..660 TFLOP/s), 8192^2 x 16 heads of 128 575 us (955), one token against 16 x 16384 keys of 8 heads of 128 199 us with the
// join (5.4 TB/s); fp32: 2 x 4096^2 x 4 heads of 32 110 us (156 TFLOP/s), the token's three planes per key 2.6 TB/s.
#include "attention_device.h"

namespace eq {

template <int T>
struct AttnFwd {
    AttnShape s;
    AttnTensor<T> q, k, v;
    typename Num<T>::type* out;               // [batch, nq, heads, dim] contiguous
    typename Num<T>::type* out_low;           // 16-bit types, for the backward: what out's rounding dropped, or null
    float* lse;                               // [batch, kv_heads, nq * group] base-2 log-sum of the scaled scores, +inf for a row without keys, NaN for a NaN sum
    int row_tiles, splits, split_keys;
    float* part_o;                            // [splits][batch * kv_heads][nq * group][dim]
    float* part_l;                            // [splits][batch * kv_heads][nq * group], -inf for a part without keys
};

template <int T>
__device__ __forceinline__ void attn_store_out(typename Num<T>::type* out, typename Num<T>::type* low, const float (&x)[4], int n) {
    store4<T>(out, x, n);
    if (T != kF32 && low) {
        float r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = x[i] - (float)(typename Num<T>::type)x[i];
        store4<T>(low, r, n);
    }
}

// W: width of the staged tiles, KS: steps of 16 that the head dim takes in them
template <int T, int W, int KS, int NW>
__global__ __launch_bounds__(NW * 64, W == 128 && T == kF32 ? 1 : 2) void attn_fwd_kernel(AttnFwd<T> a) {
    constexpr int KT = attn_tile<T, W>(), NT = NW * 64, ROWS = NW * 32, NP = Num<T>::planes;
    constexpr int DB = (KS + 1) / 2, KB = KT / 32;
    // fp16: P is held as 2^8 P, so that probabilities down to 2^-32 count; with the slack that stays below 2^14
    constexpr float kShift = T == kF16 ? 8.f : 0.f, kSlack = T == kF16 ? 6.f : 8.f;
    __shared__ __attribute__((aligned(16))) short tile_k[NP * Tile<W>::size(KT)];
    __shared__ __attribute__((aligned(16))) short tile_v[NP * Tile<W>::size(KT)];
    __shared__ __attribute__((aligned(16))) float hidden[KT];
    const AttnShape& s = a.s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const AttnUnit un = attn_unit(s.batch * s.kv_heads, a.row_tiles * a.splits);
    const int rt = a.row_tiles - 1 - un.unit / a.splits, split = un.unit % a.splits;      // causal: the longest tiles first
    const int bh = un.bh, b = bh / s.kv_heads, hk = bh - b * s.kv_heads;
    const int ql = attn_len(s.q_lens, b, s.nq), kl = attn_len(s.kv_lens, b, s.nk);
    const int rows = s.nq * s.group, rows_valid = ql * s.group, row0 = rt * ROWS;
    const int row = row0 + wave * 32 + (lane & 31);
    int k_end = min(kl, (split + 1) * a.split_keys);
    const int k_begin = split * a.split_keys;
    const int last_row = min(row0 + ROWS, rows_valid) - 1;
    if (s.causal && last_row >= 0) k_end = min(k_end, row_point(s, last_row) + kl - ql + 1);
    if (row0 >= rows_valid) k_end = 0;
    const int limit = s.causal ? row_point(s, row) + kl - ql : 0x7fffffff;      // this lane's last visible key
    const uint8_t* mask = s.key_mask ? s.key_mask + b * s.mask_stride : nullptr;

    Op8<T> q[KS];
    {
        const bool ok = row < rows_valid;
        const typename Num<T>::type* p = ok ? packed_row(a.q, s, b, hk, row) : nullptr;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) q[ks] = planes_of<T>(ok ? load8<T>(p, ks * 16 + half * 8, s.dim) : raw_zero<T>());
    }
    pf32x16 acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
    float m = -INFINITY, l = 0.f;

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
        __syncthreads();                                  // the previous tile has been read
        sk.store(tile_k);
        sv.store(tile_v);
        if (threadIdx.x < KT) hidden[threadIdx.x] = vis ? 0.f : 1.f;
        __syncthreads();
        if (k0 + KT < k_end) load_tile(k0 + KT);
        pf32x16 sc[KB];
        __builtin_amdgcn_s_setprio(1);                    // a wave with products to issue goes before one in its softmax
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[kb][r] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) mma<T>(sc[kb], tile_rows<T, W, KT>(tile_k, kb * 32, ks, lane), q[ks]);
        }
        __builtin_amdgcn_s_setprio(0);
        const bool edge = mask || k0 + KT > k_end || (s.causal && k0 + KT > row_point(s, row0 + wave * 32) + kl - ql + 1);
        if (edge) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int j = kb * 32 + 8 * g + 4 * half;
                    const pf32x4 h = *reinterpret_cast<const pf32x4*>(hidden + j);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (h[i] != 0.f || k0 + j + i > limit) sc[kb][4 * g + i] = -INFINITY;
                }
        }
        float top = sc[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, sc[kb][r]);
        // The reference value m only has to keep the exponentials in range: it follows the running maximum when that has risen by more
        // than 2^kSlack, which is rare after the first tiles, and the accumulators are rescaled only then.
        if (__any((top - m) * s.scale_log2 > kSlack)) {       // (-inf) - (-inf) is NaN: no
            top = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
            const float old = top == -INFINITY ? 1.f : exp2_fast((m - top) * s.scale_log2);
            m = top;
            l *= old;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= old;
        }
        const float sub = m == -INFINITY ? 0.f : kShift - m * s.scale_log2;      // nothing visible so far: exp2(-inf) = 0
        float sum = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                sc[kb][r] = exp2_fast(fmaf(sc[kb][r], s.scale_log2, sub));
                sum += sc[kb][r];
            }
        l += sum;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = sc[kb][8 * t + j];
                const Op8<T> p = pack8<T>(x);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const Op8<T> v = tile_cols<T, W, KT>(tile_v, kb * 32 + 16 * t, d * 32, lane);
                    if constexpr (attn_two_planes<T, KS>()) mma<T>(acc[d], v, pack8_rest<T>(x));
                    mma<T>(acc[d], v, p);
                }
            }
    }
    if (row >= rows) return;
    l += __shfl_xor(l, 32);
    const bool exists = row < rows_valid;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // a NaN sum stays NaN, an empty row becomes zero
    // a row without keys: +inf (its probabilities are zero); a NaN sum stays NaN, so that the backward's probabilities are NaN for all its keys
    const float lse = !exists || l == 0.f ? INFINITY : fmaf(m, s.scale_log2, log2f(l) - kShift);
    const int64_t at = (int64_t)bh * rows + row;
    if (a.splits > 1) {
        const int64_t pat = ((int64_t)split * s.batch * s.kv_heads + bh) * rows + row;
        if (half == 0) a.part_l[pat] = lse == INFINITY ? -INFINITY : lse;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = d * 32 + 8 * g + 4 * half;
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = exists ? acc[d][4 * g + i] * inv : 0.f;
                store4<kF32>(a.part_o + pat * s.dim + c, x, s.dim - c);
            }
        return;
    }
    if (a.lse && half == 0) a.lse[at] = lse;
    const int i0 = row_point(s, row);
    const int64_t o = (((int64_t)b * s.nq + i0) * s.heads + hk * s.group + row - i0 * s.group) * s.dim;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = d * 32 + 8 * g + 4 * half;
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = exists ? acc[d][4 * g + i] * inv : 0.f;
            attn_store_out<T>(a.out + o + c, a.out_low ? a.out_low + o + c : nullptr, x, s.dim - c);
        }
}

// joins the parts of a split key axis, in split order: a thread per four values of a row
template <int T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnFwd<T> a) {
    const AttnShape& s = a.s;
    const int rows = s.nq * s.group, quads = (s.dim + 3) / 4;
    const int64_t n = (int64_t)s.batch * s.kv_heads * rows, id = (int64_t)blockIdx.x * 256 + threadIdx.x, at = id / quads;
    if (at >= n) return;
    const int c = (int)(id - at * quads) * 4, left = min(4, s.dim - c);
    const int bh = (int)(at / rows), row = (int)(at - (int64_t)bh * rows), b = bh / s.kv_heads, hk = bh - b * s.kv_heads;
    float top = -INFINITY;
    for (int i = 0; i < a.splits; ++i) top = fmaxf(top, a.part_l[i * n + at]);
    const float use = top == -INFINITY ? 0.f : top;
    float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < a.splits; ++i) {
        const float w = exp2_fast(a.part_l[i * n + at] - use);
        const float* p = a.part_o + (i * n + at) * s.dim + c;
        sum += w;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < left) v[e] = fmaf(w, p[e], v[e]);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (a.lse && c == 0) a.lse[at] = sum == 0.f ? INFINITY : use + log2f(sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= inv;
    const int i0 = row_point(s, row);
    const int64_t o = (((int64_t)b * s.nq + i0) * s.heads + hk * s.group + row - i0 * s.group) * s.dim + c;
    attn_store_out<T>(a.out + o, a.out_low ? a.out_low + o : nullptr, v, left);
}

// Rows of a workgroup: 128 (four waves share every key tile), or 32 when there are no more rows than that per key head (single tokens).
// Splits: the key axis is cut when the row tiles alone leave compute units idle, into parts of whole key tiles, one part for every four tiles
// at most (a length just above a multiple of four tiles gives parts of three, and the last part takes what is left).  fp32 heads of 32: 4 tokens against
// 16384 keys of 8 heads 68 us (117 with parts of two tiles: the join reads twice as many), one token against 1000 keys of 2 heads 23 (21).
struct AttnPlan { int waves, row_tiles, splits, split_keys; };
static AttnPlan attn_plan(int dtype, const AttnShape& s) {
    const int rows = s.nq * s.group, nk = s.nk, kt = attn_tile_of(dtype, s.dim);
    AttnPlan p;
    p.waves = rows <= 32 ? 1 : 4;
    p.row_tiles = ceil_div(rows, p.waves * 32);
    const int64_t blocks = (int64_t)p.row_tiles * s.batch * s.kv_heads, want = p.waves == 1 ? 1024 : 512;
    const int most = ceil_div(nk, 4 * kt);
    p.splits = 1;
    if (blocks * 2 <= want && most > 1) p.splits = (int)(want / blocks < most ? want / blocks : most);
    p.split_keys = ceil_div(ceil_div(nk, p.splits), kt) * kt;
    p.splits = nk > 0 ? ceil_div(nk, p.split_keys) : 1;
    return p;
}

template <int T, int W, int KS>
static int attn_fwd_launch(const AttnFwd<T>& a, int waves, int64_t blocks, hipStream_t st) {
    if (waves == 1) attn_fwd_kernel<T, W, KS, 1><<<(unsigned)blocks, 64, 0, st>>>(a);
    else attn_fwd_kernel<T, W, KS, 4><<<(unsigned)blocks, 256, 0, st>>>(a);
    EQ_CHECK_LAUNCH("attention_forward");
    return 0;
}

template <int T>
static int attn_fwd(const equigspr_attention* d, const AttnShape& s, void* out, void* out_low, float* lse, float* work, hipStream_t st) {
    using E = typename Num<T>::type;
    AttnFwd<T> a;
    a.s = s;
    a.q = attn_tensor<T>(d->q, s.dim);
    a.k = attn_tensor<T>(d->k, s.dim);
    a.v = attn_tensor<T>(d->v, s.dim);
    a.out = (E*)out;
    a.out_low = (E*)out_low;
    a.lse = lse;
    const AttnPlan p = attn_plan(T, s);
    a.row_tiles = p.row_tiles; a.splits = p.splits; a.split_keys = p.split_keys;
    const int64_t n = (int64_t)s.batch * s.kv_heads * s.nq * s.group;
    a.part_l = work;
    a.part_o = work + (p.splits > 1 ? (p.splits * n + 3) / 4 * 4 : 0);
    const int64_t blocks = (int64_t)p.row_tiles * p.splits * s.batch * s.kv_heads;
    EQ_CHECK_ARG(blocks < (1 << 24), EQUIGSPR_ENOTSUP, "attention: %lld workgroups are more than one launch takes", (long long)blocks);
    const int rc = EQ_ATTN_BY_DIM(attn_fwd_launch, s.dim, a, p.waves, blocks, st);
    if (rc || p.splits == 1) return rc;
    attn_join_kernel<T><<<(unsigned)ceil_div(n * ((s.dim + 3) / 4), 256), 256, 0, st>>>(a);
    EQ_CHECK_LAUNCH("attention_forward (join)");
    return 0;
}

int attn_shape(const equigspr_attention* d, AttnShape* s) {
    EQ_CHECK_ARG(d, EQUIGSPR_EINVAL, "attention: null description");
    EQ_CHECK_ARG(d->dtype == EQUIGSPR_F32 || d->dtype == EQUIGSPR_BF16 || d->dtype == EQUIGSPR_F16, EQUIGSPR_EINVAL, "attention: unknown dtype %d", d->dtype);
    EQ_CHECK_ARG(d->batch >= 0 && d->nq >= 0 && d->nk >= 0 && d->heads >= 1 && d->kv_heads >= 1, EQUIGSPR_EINVAL, "attention: negative size");
    EQ_CHECK_ARG(d->heads % d->kv_heads == 0, EQUIGSPR_EINVAL, "attention: %d heads are not a multiple of %d key heads", d->heads, d->kv_heads);
    EQ_CHECK_ARG(d->dim >= 1 && d->dim <= kAttnMaxDim, EQUIGSPR_ENOTSUP, "attention: head dim %d, the kernels take 1..%d", d->dim, kAttnMaxDim);
    EQ_CHECK_ARG(d->scale > 0.f && d->scale < INFINITY, EQUIGSPR_EINVAL, "attention: the scale must be positive and finite");
    const int64_t g = d->heads / d->kv_heads;
    EQ_CHECK_ARG(d->nq * g * g < (1ll << 32) && d->nq * g < (1ll << 30) && d->nk < (1 << 30) && (int64_t)d->batch * d->heads < (1 << 24), EQUIGSPR_ENOTSUP,
                 "attention: too many rows, keys or heads for one call");
    const int esize = d->dtype == EQUIGSPR_F32 ? 4 : 2;
    EQ_CHECK_ARG(attn_near(d->q, esize) && attn_near(d->k, esize) && attn_near(d->v, esize), EQUIGSPR_ENOTSUP,
                 "attention: negative strides, or points or heads further apart than 2^31 / 128 bytes");
    EQ_CHECK_ARG(!d->batch || ((d->q.data || !d->nq) && ((d->k.data && d->v.data) || !d->nk)), EQUIGSPR_EINVAL, "attention: null tensor");
    s->batch = d->batch; s->nq = d->nq; s->nk = d->nk; s->heads = d->heads; s->kv_heads = d->kv_heads; s->group = (int)g; s->dim = d->dim;
    s->group_magic = (unsigned)(((1ull << 32) + g - 1) / g);
    s->scale = d->scale;
    s->scale_log2 = d->scale * 1.4426950408889634f;
    s->causal = d->causal != 0;
    s->q_lens = d->q_lens; s->kv_lens = d->kv_lens; s->key_mask = d->key_mask; s->mask_stride = d->mask_stride;
    return 0;
}

}  // namespace eq

extern "C" int64_t equigspr_attention_work_size(const equigspr_attention* d) {
    eq::AttnShape s;
    if (eq::attn_shape(d, &s) != 0) return -1;
    const eq::AttnPlan p = eq::attn_plan(d->dtype, s);
    if (p.splits == 1) return 0;
    const int64_t n = (int64_t)s.batch * s.kv_heads * s.nq * s.group;
    return (p.splits * n + 3) / 4 * 4 + p.splits * n * s.dim;
}

extern "C" int equigspr_attention_forward(const equigspr_attention* d, void* out, void* out_low, float* lse, float* work, void* stream) {
    eq::AttnShape s;
    if (const int rc = eq::attn_shape(d, &s)) return rc;
    EQ_CHECK_ARG(out || !s.batch || !s.nq, EQUIGSPR_EINVAL, "attention_forward: out is null");
    EQ_CHECK_ARG(work || equigspr_attention_work_size(d) == 0, EQUIGSPR_EINVAL, "attention_forward: work is null");
    if (s.batch == 0 || s.nq == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    switch (d->dtype) {
        case EQUIGSPR_F32: return eq::attn_fwd<eq::kF32>(d, s, out, out_low, lse, work, st);
        case EQUIGSPR_BF16: return eq::attn_fwd<eq::kBF16>(d, s, out, out_low, lse, work, st);
        default: return eq::attn_fwd<eq::kF16>(d, s, out, out_low, lse, work, st);
    }
}
