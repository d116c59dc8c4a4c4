// Decode attention over pages: arguments, the split of the work and the memory-bound kernel.
//
//   o = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),   s_t = scale <q, k_hat_t>,   m = max_t s_t
//
// Work is an ordered list of tiles of kTile tokens: for each KV head, each sequence and each 16 query rows of
// it (an item), the item's tiles.  The list is cut into equal ranges, one per CTA of a persistent grid, so
// that ragged lengths balance and a CTA changes its head's codebook at most a few times.  A range holds whole
// items, which are finished in place, and at most two cut ones, whose (m, l, acc) go to workspace slots that a
// second kernel joins in a fixed order.
#pragma once

#include <cudaTypedefs.h>

#include "paged.cuh"

namespace sunshape {

constexpr int kTile = 32;          // tokens of a tile, consumed by one warp
constexpr int kItemRows = 16;      // query rows of an item: the M of one MMA
constexpr int kConsumers = 8;      // consumer warps, two warpgroups
constexpr int kProducers = 4;      // producer warps, one warpgroup
constexpr int kAttnThreads = (kConsumers + kProducers) * 32;
// Registers of a thread: what the block is launched with, and its split between the roles (setmaxnreg).
constexpr int kLaunchRegs = 168, kConsumerRegs = 216, kProducerRegs = 72;
static_assert(kConsumers * kConsumerRegs + kProducers * kProducerRegs <= (kConsumers + kProducers) * kLaunchRegs, "");
constexpr int kPlanChunks = 256;   // sequence chunks of the in-kernel plan

struct AttnParams {
  const void* q;
  int64_t qs[3];                   // strides of (b, h, l), elements
  int B, Hq, H, L, G, nb, n_cb, ps, n_heavy, cols, causal, stages, stage_bytes, off_idx, off_heavy;
  int chunk;                       // tokens of a copy: 32, or 16 where pages are no multiple of 32
  int prefix_mode;                 // 1: the one sequence is the prefix, rows are those of all sequences
  int prefix_len;
  int prefix_parts;                // partial sets of the prefix that a finished row joins (0: none)
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
  float* slots;                    // [2 * grid][kItemRows][2 + DV] cut items
  int4* desc;                      // [grid] (head piece: 0 none, 1 cut again, 2 last; tail item h, b, row tile) -- h -1: none
  float* prefix_part;              // [prefix_parts][B * Hq * L][2 + DV]
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

// Finished rows: out = acc / l, joined with the prefix's partial sets where there are any.
template <typename T, int DV>
__device__ __forceinline__ void finish_element(const AttnParams& p, const RowMap& at, int d, float m, float l, float a) {
  const int64_t row = ((int64_t)at.b * p.Hq + at.hq) * p.L + at.l;
  if (p.prefix_mode) {
    float* dst = p.prefix_part + row * (DV + 2);
    dst[2 + d] = a;
    if (d == 0) {
      dst[0] = m;
      dst[1] = l;
    }
    return;
  }
  const float INF = __int_as_float(0x7f800000);
  if (p.prefix_parts) {
    const int64_t rows = (int64_t)p.B * p.Hq * p.L;
    float M = m;
    for (int k = 0; k < p.prefix_parts; ++k) M = fmaxf(M, p.prefix_part[(k * rows + row) * (DV + 2)]);
    const float base = M == -INF ? 0.f : M;
    float f = fast_exp2(m - base);
    l *= f;
    a *= f;
    for (int k = 0; k < p.prefix_parts; ++k) {
      const float* src = p.prefix_part + (k * rows + row) * (DV + 2);
      f = fast_exp2(src[0] - base);
      l = fmaf(src[1], f, l);
      a = fmaf(src[2 + d], f, a);
    }
  }
  // l is 0 only where the row saw no token
  reinterpret_cast<T*>(p.out)[row * DV + d] = Elem<T>::from_float(l == 0.f ? 0.f : a / l);
}

template <int D, int DV, int BD, typename T>
int launch_paged_attention(const AttnParams& p, const CUtensorMap& vmap, int grid, cudaStream_t st);

}  // namespace sunshape
