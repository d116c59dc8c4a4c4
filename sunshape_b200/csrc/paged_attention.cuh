// Decode attention over pages: arguments, the split of the work and what finishes a row.
//
//   o = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),   s_t = scale <q, k_hat_t>,   m = max_t s_t
//
// Work is an ordered list of tiles of kTile tokens: for each KV head, each sequence and each group of query rows
// of it (an item), the item's tiles.  The list is cut into equal ranges, one per CTA of a persistent grid, and a
// CTA's range into equal ranges, one per pair of a producer and a consumer warp, so that ragged lengths balance
// and no warp waits for another before its range is done.  A pair finishes the items that lie whole in its range;
// those cut between pairs are joined in shared memory when the CTA's range ends, those cut between CTAs go as
// (m, l, acc) to workspace slots that a second kernel joins.  Every join takes the pieces in the list's order, so
// results do not depend on timing.
#pragma once

#include <cudaTypedefs.h>

#include "paged.cuh"

namespace sunshape {

constexpr int kSmemMax = 232448;   // 227 KB
constexpr int kTile = 32;          // tokens of a tile
constexpr int kItemRows = 16;      // most query rows of an item
constexpr int kPairs = 8;          // pairs of a consumer (warps 0-7) and a producer warp (8-15)
constexpr int kAttnThreads = 2 * kPairs * 32;
constexpr int kMinTiles = kPairs;  // tiles of a CTA's range, unless there are fewer: one for each pair
// Tiles that other work is charged in the split.  The change to another head's codebook (the pairs drain, 64 KB are copied,
// queries and first tiles follow) takes a CTA about as long as 50 tiles at HBM's pace: 64 sequences of 1k to 8k take 118 us
// with 16 charged, 114 with 48.
constexpr int kHeadTiles = 48;
// The queries and the result of an item of 16 rows (16 sequences of 3 to 6k, 4 queries: 64 us with 2, 54 with 5, 53 with
// 14); of 8 rows, 2 (64 sequences of up to 700 tokens, 64/8 heads: 28.9 us with 0, 25.7 with 2).
constexpr int kItemTiles = 5;
constexpr int kPlanChunks = 256;   // sequence chunks of the in-kernel plan
// Registers of a thread: what the block is launched with, and its split between the roles (setmaxnreg).  Not enough for either:
// at D = DV = 128 the compiler spills 148 to 200 bytes a thread with one group of eight rows and 516 to 612 with two, whose
// consumer holds 2 x 32 accumulators, 2 x 16 words of queries and a tile's keys.
constexpr int kLaunchRegs = 128, kConsumerRegs = 216, kProducerRegs = 40;
static_assert(kConsumerRegs + kProducerRegs <= 2 * kLaunchRegs, "the split waits forever where it exceeds the launch");

// One row of a piece or partial set: acc[DV], m (in powers of two), l, two unused.
__host__ __device__ constexpr int row_floats(int dv) { return dv + 4; }

struct AttnParams {
  const void* q;
  int64_t qs[3];                   // strides of (b, h, l), elements
  int B, Hq, H, L, G, nb, n_cb, ps, n_heavy, cols, causal, pairs, stages, stage_bytes, off_idx, off_heavy;   // stages: of a pair
  int chunk;                       // tokens of a copy: 32, or 16 where pages are no multiple of 32
  int prefix_mode;                 // 1: the one sequence is the prefix, rows are those of all sequences
  int prefix_len;
  int prefix_parts;                // partial sets of the prefix that a finished row joins (0: none)
  int overlap;                     // 1: may start before the prefix's sets are written (griddepcontrol.wait comes before them)
  int64_t num_pages, table_stride;
  float scale_log2;                // scale * log2(e)
  const int32_t* table;
  const int32_t* lens;
  const int64_t* perm;
  const uint8_t* heavy_mask;
  const uint8_t* idx;
  const void* heavy;
  const void* image;               // fp16 codebooks
  const float* image_scale;
  void* out;
  float* slots;                    // [2 * grid][kItemRows] rows: pieces of items cut between CTAs
  int4* desc;                      // [grid] (head piece: 0 none, 1 cut again, 2 last; tail item's h (-1: none), b, row group)
  float* pieces;                   // [grid][kPairs][2][item_rows] rows: pieces of items cut between a CTA's pairs
  float* prefix_part;              // [prefix_parts][B * Hq * L] rows
  float* prefix_slots;             // [2 * grid][256] rows: pieces of the prefix's items cut between CTAs
  int* err;
  int item_rows;                   // 8 or 16: which kernel
  int smem;
};

// capi.cu
int make_rows_map(CUtensorMap* map, const void* base, bool bf16, int cols, int64_t rows, int box_rows);

// Rows of an item: number and, per row, the sequence, query head and query token.
struct RowMap {
  int b, hq, l;
};

__device__ __forceinline__ int item_rows_total(const AttnParams& p) {
  return p.prefix_mode ? p.B * p.G * p.L : p.G * p.L;
}

__device__ __forceinline__ RowMap row_of(const AttnParams& p, int h, int b, int r) {
  if (p.prefix_mode) {
    b = r / (p.G * p.L);
    r -= b * p.G * p.L;
  }
  const int g = r / p.L;
  return {b, h * p.G + g, r - g * p.L};
}

// A sequence's own length, -1 where it does not fit its table.
__device__ __forceinline__ int own_length(const AttnParams& p, int b) {
  if (p.prefix_mode) return p.prefix_len;
  const int n = p.lens[b];
  return n < 0 || n > (int64_t)p.cols * p.ps ? -1 : n;
}

// tiles of a sequence: at least one, so that empty sequences are written too
__device__ __forceinline__ int tiles_of(int len) { return len <= 0 ? 1 : (len + kTile - 1) / kTile; }

// Index of a row in out and in the prefix's partial sets.
__device__ __forceinline__ int64_t flat_row(const AttnParams& p, const RowMap& at) {
  return ((int64_t)at.b * p.Hq + at.hq) * p.L + at.l;
}

// What a finished row does with its accumulators: out = (f acc + sum over the prefix's sets of fk acck) / l.
struct Finish {
  float f, inv;        // factor of the row's own acc, 1 / l
  float base;          // the maximum that factors refer to
};

template <int DV>
__device__ __forceinline__ Finish finish_of(const AttnParams& p, int64_t row, float m, float l) {
  const float INF = __int_as_float(0x7f800000);
  float top = m;
  const int64_t rows = (int64_t)p.B * p.Hq * p.L;
  for (int k = 0; k < p.prefix_parts; ++k)
    top = fmaxf(top, p.prefix_part[(k * rows + row) * row_floats(DV) + DV]);
  Finish e;
  e.base = top == -INF ? 0.f : top;
  e.f = fast_exp2(m - e.base);
  l *= e.f;
  for (int k = 0; k < p.prefix_parts; ++k) {
    const float* src = p.prefix_part + (k * rows + row) * row_floats(DV) + DV;
    l = fmaf(src[1], fast_exp2(src[0] - e.base), l);
  }
  e.inv = l == 0.f ? 0.f : 1.f / l;      // l is 0 only where the row saw no token
  return e;
}

// Of a row of a codec with dense blocks whose sum is no number: records it, unless that is the query's doing.
template <int D, typename T>
__device__ __forceinline__ void report_dense(const AttnParams& p, const RowMap& at) {
  const T* q = reinterpret_cast<const T*>(p.q) + at.b * p.qs[0] + at.hq * p.qs[1] + at.l * p.qs[2];
#pragma unroll 1
  for (int d = 0; d < D; ++d)
    if (!(fabsf(Elem<T>::to_float(q[d])) < __int_as_float(0x7f800000))) return;
  record_error(p.err, kErrDense);
}

// Four columns of a row.
template <typename T, int DV>
__device__ __forceinline__ void finish4(const AttnParams& p, const RowMap& at, int d, float m, float l, float4 a) {
  const int64_t row = flat_row(p, at);
  if (p.prefix_mode) {
    float* dst = p.prefix_part + row * row_floats(DV);
    *reinterpret_cast<float4*>(dst + d) = a;
    if (d == 0) *reinterpret_cast<float2*>(dst + DV) = make_float2(m, l);
    return;
  }
  const Finish e = finish_of<DV>(p, row, m, l);
  a = make_float4(a.x * e.f, a.y * e.f, a.z * e.f, a.w * e.f);
  const int64_t rows = (int64_t)p.B * p.Hq * p.L;
  for (int k = 0; k < p.prefix_parts; ++k) {
    const float* src = p.prefix_part + (k * rows + row) * row_floats(DV);
    const float f = fast_exp2(src[DV] - e.base);
    const float4 b = *reinterpret_cast<const float4*>(src + d);
    a = make_float4(fmaf(b.x, f, a.x), fmaf(b.y, f, a.y), fmaf(b.z, f, a.z), fmaf(b.w, f, a.w));
  }
  T r[4] = {Elem<T>::from_float(a.x * e.inv), Elem<T>::from_float(a.y * e.inv), Elem<T>::from_float(a.z * e.inv),
            Elem<T>::from_float(a.w * e.inv)};
  *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + row * DV + d) = *reinterpret_cast<const uint2*>(r);
}

// Adds a piece (mk, lk, ak) that follows (m, l, a) in the list.
__device__ __forceinline__ void join4(float& m, float& l, float4& a, float mk, float lk, float4 ak) {
  const float INF = __int_as_float(0x7f800000);
  const float top = fmaxf(m, mk), base = top == -INF ? 0.f : top;
  const float f = fast_exp2(m - base), fk = fast_exp2(mk - base);
  l = l * f + lk * fk;
  a = make_float4(a.x * f + ak.x * fk, a.y * f + ak.y * fk, a.z * f + ak.z * fk, a.w * f + ak.w * fk);
  m = top;
}

template <int D, int DV, int BD, typename T>
int launch_paged_attention(const AttnParams& p, const CUtensorMap& vmap, int grid, cudaStream_t st);
template <int D, int DV, int BD, typename T>
int launch_paged_prefix(const AttnParams& p, const CUtensorMap& vmap, int grid, cudaStream_t st);

}  // namespace sunshape
