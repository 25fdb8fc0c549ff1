// What the attention kernels (attention.hip, attention_bwd.hip) share: the problem's description, the packed row order, the staging
// of rows into LDS tiles.
//
// Rows are PACKED: the G = heads / kv_heads query heads that share a key head form one row axis, row r = i G + g of point i and head
// g of the group.  A key tile is then read once for the whole group, and the gradients of the shared keys are summed inside one
// workgroup, in a fixed order.
#pragma once
#include "planes.h"

namespace eq {

struct AttnShape {
    int batch, nq, nk, heads, kv_heads, group, dim;
    unsigned group_magic;                     // ceil(2^32 / group): r / group = umulhi(r, magic) while rows * group < 2^32 (host check)
    float scale_log2;                         // scale * log2(e)
    float scale;
    int causal;
    const int32_t* q_lens;                    // [batch] or null
    const int32_t* kv_lens;
    const uint8_t* key_mask;                  // [batch, nk] or null, non-zero = visible
    int64_t mask_stride;
};

// [batch, points, heads, dim] with unit stride in dim
template <int T>
struct AttnTensor {
    typename Num<T>::type* p;
    int64_t sb, sn, sh;
};

__device__ __forceinline__ int attn_len(const int32_t* lens, int b, int n) {
    if (!lens) return n;
    const int v = lens[b];
    return v < 0 ? 0 : (v > n ? n : v);
}
__device__ __forceinline__ int row_point(const AttnShape& s, int r) { return s.group == 1 ? r : (int)__umulhi((unsigned)r, s.group_magic); }

template <int T>
__device__ __forceinline__ typename Num<T>::type* packed_row(const AttnTensor<T>& t, const AttnShape& s, int b, int hk, int r) {
    const int i = row_point(s, r), g = r - i * s.group;
    return t.p + b * t.sb + i * t.sn + (int64_t)(hk * s.group + g) * t.sh;
}
template <int T>
__device__ __forceinline__ typename Num<T>::type* key_row(const AttnTensor<T>& t, int b, int hk, int j) {
    return t.p + b * t.sb + j * t.sn + (int64_t)hk * t.sh;
}

// ROWS x W values from memory to the planes of a tile by NT threads: load() to registers, store() to LDS, so that the next tile's
// loads are in flight under this tile's products.  A thread's chunks all lie in one column of chunks.
template <int T, int W, int ROWS, int NT>
struct Stager {
    using E = typename Num<T>::type;
    static constexpr int kChunks = W / 8, kPer = ROWS * kChunks / NT, kPlane = Tile<W>::size(ROWS);      // chunks of a row, of a thread; values of a plane
    static_assert(kPer * NT == ROWS * kChunks && NT % kChunks == 0, "whole chunks per thread");
    Raw8<T> raw[kPer];
    unsigned off[kPer];                       // of the thread's chunks from the tile's first row, when rows lie at fixed distances
    // row_off(r): distance of row r of a tile from its first row, in values, below 2^31 bytes (host check)
    template <class F>
    __device__ __forceinline__ void init(F row_off) {
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            const int id = threadIdx.x + u * NT;
            off[u] = (unsigned)((row_off(id / kChunks) + (id % kChunks) * 8) * (int)sizeof(E));
        }
    }
    // a whole tile of existing rows, width % 8 == 0: one base in scalar registers, the threads' offsets computed once
    __device__ __forceinline__ void load_whole(const E* first_row, int width) {
        const bool in = (int)(threadIdx.x % kChunks) * 8 < width;
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            if (!in) raw[u] = raw_zero<T>();
            else raw[u] = load8<T>(reinterpret_cast<const E*>(reinterpret_cast<const char*>(first_row) + off[u]), 0, 8);
        }
    }
    // row_of(r) -> pointer of row r, or null for a row of zeros
    template <class F>
    __device__ __forceinline__ void load(F row_of, int width) {
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            const int id = threadIdx.x + u * NT;
            const E* row = row_of(id / kChunks);
            raw[u] = row ? load8<T>(row, (id % kChunks) * 8, width) : raw_zero<T>();
        }
    }
    __device__ __forceinline__ void store(short* tile) const {
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            const int id = threadIdx.x + u * NT;
            const Op8<T> o = planes_of<T>(raw[u]);
#pragma unroll
            for (int p = 0; p < Num<T>::planes; ++p)
                *reinterpret_cast<s16x8*>(tile + p * kPlane + Tile<W>::at(id / kChunks, id % kChunks)) = o.p[p];
        }
    }
};

// A operand: 32 rows of the tile from row0, k-step ks (16 columns)
template <int T, int W, int ROWS>
__device__ __forceinline__ Op8<T> tile_rows(const short* tile, int row0, int ks, int lane) {
    Op8<T> o;
#pragma unroll
    for (int p = 0; p < Num<T>::planes; ++p) o.p[p] = Tile<W>::row8(tile + p * Tile<W>::size(ROWS), row0 + (lane & 31), 2 * ks + (lane >> 5));
    return o;
}
// A operand of the transposed tile: 32 columns from col0 as rows; the contraction runs over the 16 tile rows from row0 in the order in
// which the C tile of an earlier product holds them (slot j of half h is row 8 (j >> 2) + 4 h + (j & 3)), so that product's result is
// the B operand as it stands
template <int T, int W, int ROWS>
__device__ __forceinline__ Op8<T> tile_cols(const short* tile, int row0, int col0, int lane) {
    Op8<T> o;
    const int r = row0 + 4 * (lane >> 5), c = col0 + (lane & 16);
#pragma unroll
    for (int p = 0; p < Num<T>::planes; ++p)
        o.p[p] = join8(Tile<W>::col4(tile + p * Tile<W>::size(ROWS), r, c, lane), Tile<W>::col4(tile + p * Tile<W>::size(ROWS), r + 8, c, lane));
    return o;
}

// Which head and which of its `units` (tiles, longest first) a workgroup takes.  Workgroups are dealt to the eight XCDs in turn, so with
// the head running fastest an XCD sees the same few heads again and again (their keys stay in its L2) and every XCD sees every sample --
// lengths differ between samples, so a contiguous run of heads per XCD left some idle (8 ragged samples of 2048 points, 8 heads of 64: forward 113 us
// against 100, keys' gradients 320 against 170).  Heads are taken
// 32 at a time, so that no more than four heads' keys pass through an XCD at once.
struct AttnUnit { int bh, unit; };
__device__ __forceinline__ AttnUnit attn_unit(int heads, int units) {
    const int per = 32 * units, group = blockIdx.x / per, r = blockIdx.x - group * per, n = min(32, heads - 32 * group);
    return {32 * group + r % n, r / n};
}

// 16-bit heads of up to 16 dims: P and dS enter their products in two planes.  Their rounding hardly averages out there (gradients of q 1.6
// times as far off as the plain form's, 1.4 for wider heads), and the second product is one matrix instruction.
template <int T, int KS> constexpr bool attn_two_planes() { return T != kF32 && KS == 1; }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr int kAttnMaxDim = 128;

// rows of a staged tile: 64, except where three planes of a wide head would take too much LDS
template <int T, int W> constexpr int attn_tile() { return T == kF32 && W > 32 ? 32 : 64; }
// the same for a head dim, on the host (W is 32 up to 32 dims)
static inline int attn_tile_of(int dtype, int dim) { return dtype == kF32 && dim > 32 ? 32 : 64; }

// ---- host side
// f<T, W, KS>: the head dim in steps of 16, in tiles of 32, 64 or 128 columns (dims up to 16 and up to 96 skip the empty steps)
#define EQ_ATTN_BY_DIM(f, dim, ...)                                                                               \
    ((dim) <= 16 ? f<T, 32, 1>(__VA_ARGS__) : (dim) <= 32 ? f<T, 32, 2>(__VA_ARGS__) : (dim) <= 64 ? f<T, 64, 4>(__VA_ARGS__) \
     : (dim) <= 96 ? f<T, 128, 6>(__VA_ARGS__) : f<T, 128, 8>(__VA_ARGS__))

template <int T>
static inline AttnTensor<T> attn_tensor(const equigspr_attention_tensor& t, int dim) {
    using E = typename Num<T>::type;
    AttnTensor<T> r;
    r.p = (E*)t.data;
    r.sb = t.stride_batch; r.sn = t.stride_point; r.sh = t.stride_head;
    return r;
}

// rows of a tile lie within 2^31 bytes of each other (the kernels' 32-bit offsets inside a tile)
static inline bool attn_near(const equigspr_attention_tensor& t, int esize) {
    const int64_t most = 1ll << 31;           // of each first: the sum must not wrap around
    if (t.stride_batch < 0 || t.stride_point < 0 || t.stride_head < 0 || t.stride_point >= most || t.stride_head >= most) return false;
    return (t.stride_point + t.stride_head) * 128 * esize < most;
}

// checks the description and derives what the kernels use; 0 or an error code
int attn_shape(const equigspr_attention* d, AttnShape* s);

}  // namespace eq
