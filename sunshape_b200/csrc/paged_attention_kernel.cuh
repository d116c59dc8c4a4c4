// The memory-bound kernel of paged attention (few query rows per KV head).
//
// Bound by HBM: a token and KV head cost n_blocks + 2 DV bytes (+ dense blocks).  Each producer warp keeps its
// consumer's ring of tiles in flight (values by TMA with the 128-byte swizzle, index and dense-block rows by bulk
// copies, page by page); one producer per consumer, since one warp takes about 670 cycles to look up, wait for and
// issue a tile, and HBM delivers one to an SM in 380.  A pair's ring is its own, so a wait for a parity can not
// pass a turn too early.
//
// Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that the few query rows are the N of the
// MMA (8 or 16 of them) and the 32 tokens fill its M.
// S^T multiplies rebuilt keys that never leave registers: the contraction's order is free, so lane t of a quad takes
// whole codewords of the blocks 4u + t -- one shared-memory load of 2 BD bytes from the head's codebook gives the
// A operand of BD / 4 MMA steps, and Q is laid out to match once per item.  Each block's codewords lie in one
// column of the shared-memory banks, and the tokens that share a load phase walk the columns in rotated order, so
// the random gathers are free of bank conflicts; a barrel of selects puts the registers back in order.
// Measured on B200, head_dim 128, 16 blocks of 8, bf16: 8 sequences of 130k tokens, 64/8 heads: 342 us (2.27 GB, 6.6 TB/s); 64
// sequences of 1k to 8k, 32/8 heads: 114 us (5.6 TB/s); a call of one tile a head 12 us, which is plan, codebook, queries,
// one tile and the join.
// P^T comes from the accumulators of S^T by a register transpose (movmatrix).
//
// What is rounded: codewords to fp16 (a second term of them would double the codebook in shared memory and halve the ring),
// queries to fp16 in a scale of the row's own (exact but for elements below 2^-14 of its largest), weights to the cache's type
// (the MMA multiplies equal types).  Scores, maxima, sums and accumulators are fp32.  On 517 tokens in f16 the result is off
// by 4e-4 where its own rounding alone is 2e-4, on 1k to 8k tokens in bf16 by 2.3e-3 against 1.7e-3.
#pragma once

#include <type_traits>
#include <utility>

#include "paged_attention.cuh"

namespace sunshape {

__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ void mma_pv(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value) {
    mma_f16(c, a0, a1, a2, a3, b0, b1);
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// transposes an 8x8 matrix of 16-bit elements held as one MMA fragment register
__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// the address is addr + OFF, folded into the instruction
template <int OFF>
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4+%5];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr), "n"(OFF));
}

template <int BYTES, int OFF>
__device__ __forceinline__ void lds_words(uint32_t* w, uint32_t addr) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4+%5];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(addr), "n"(OFF));
  else if constexpr (BYTES == 8)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2+%3];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr), "n"(OFF));
  else
    asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(w[0]) : "r"(addr), "n"(OFF));
}

// f(Index<0>()), ..., f(Index<N - 1>()): loops whose counter is a constant expression
template <int I>
struct Index {
  static constexpr int v = I;
};
template <int... I, typename F>
__device__ __forceinline__ void unrolled(std::integer_sequence<int, I...>, F&& f) {
  (f(Index<I>()), ...);
}
template <int N, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
  unrolled(std::make_integer_sequence<int, N>(), f);
}

// Dense block words (two 16-bit elements each) into the codebook's fp16 scale, a power of two of at most 1: no number of
// fp16 grows.  What bf16 has beyond fp16's 65504 becomes NaN, since an infinity would turn into a plausible result where its
// products have one sign.
template <typename T>
struct DenseScale {
  uint64_t s;
  __device__ __forceinline__ explicit DenseScale(float v) {
    const float2 two = make_float2(v, v);
    s = reinterpret_cast<const uint64_t&>(two);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t w) const {
    float2 v = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(reinterpret_cast<uint64_t&>(v)) : "l"(s));
    uint32_t r = pack2<__half>(v.x, v.y);
    asm("fma.rn.f16x2 %0, %0, %1, %0;" : "+r"(r) : "r"(0u));      // x + 0 x
    return r;
  }
};
template <>
struct DenseScale<__half> {
  uint32_t a, b;                               // in two steps, since a scale may be below fp16's numbers
  __device__ __forceinline__ explicit DenseScale(float v) {
    const float first = fmaxf(v, 6.103515625e-5f);
    a = pack2<__half>(first, first);
    b = pack2<__half>(v / first, v / first);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t w) const {
    asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(w) : "r"(a));
    asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(w) : "r"(b));
    return w;
  }
};

// A running maximum may fall behind by a factor of 2^kSlack before sums and accumulators are rescaled to a new one;
// weights stay below 2^kSlack, in reach of every type.
constexpr float kSlack = 8.f;

// Weights are 2^kShift of their share, so that fp16 drops only what is below 2^-32 of the largest (it takes numbers from
// 2^-25 to 2^16): 20000 tokens at 2^-25.5 of it each were all lost without.  bf16 reaches as far as fp32.
template <typename T>
constexpr float kShift = std::is_same<T, __half>::value ? 15.f - kSlack : 0.f;

// Where a pair stands in the list; its producer and its consumer walk it alike.
struct Walk {
  int at, end;           // tiles of the list
  int h, b, mt, t;       // the item and the tile within it
  int len, tiles;        // the sequence's length (-1: invalid) and tiles
};

// NT: groups of eight query rows of an item (1: items have at most eight rows)
template <int D, int DV, int BD, typename T, int NT>
__global__ void __launch_bounds__(kAttnThreads, 1)
    paged_attention_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap vmap) {
  constexpr int NB = D / BD, UNITS = NB / 4, WORDS = BD / 2;   // units: gathers of a lane per token
  constexpr int ROT = 16 / BD;                                 // tokens that share a load phase and a column set
  constexpr int KS = D / 16, ROWS = 8 * NT, RF = row_floats(DV);
  constexpr int IMAGE = D * 512, ITEM = NT == 1 ? 2 : kItemTiles;
  constexpr int MT = kTile / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int ring_bytes = p.stages * p.stage_bytes;             // of a pair
  uint8_t* const image = ring + (size_t)p.pairs * ring_bytes;
  int* const perm_s = reinterpret_cast<int*>(image + IMAGE);                 // [D]
  int* const len_s = perm_s + D;                                             // [kPlanChunks] lengths, where chunks are single
  int* const cum_s = len_s + kPlanChunks;                                    // [kPlanChunks + 2]
  uint64_t* const full_s = reinterpret_cast<uint64_t*>(cum_s + kPlanChunks + 2);   // [kPairs][stages]
  uint64_t* const empty_s = full_s + kPairs * p.stages;
  uint64_t* const cb_bar = empty_s + kPairs * p.stages;
  // of a pair: head piece (-1: no tiles, 0: none, 1: cut again, 2: last), its item; tail piece (0, 1), its item
  int4* const head_s = reinterpret_cast<int4*>((reinterpret_cast<uintptr_t>(cb_bar + 1) + 15) & ~uintptr_t(15));
  int4* const tail_s = head_s + kPairs;
  volatile int* const bad_s = reinterpret_cast<volatile int*>(tail_s + kPairs);    // [kPairs][stages] the tile's pages are invalid
  int8_t* const hslot_s = reinterpret_cast<int8_t*>(tail_s + kPairs) + 4 * kPairs * p.stages;   // [NB] dense slot, -1: codeword
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float INF = __int_as_float(0x7f800000);

  // ---- set-up and plan: prefix sums of tiles over chunks of sequences
  if (tid == 0) {
    for (int i = 0; i < 2 * kPairs * p.stages + 1; ++i) mbar_init(&full_s[i], 1);
    fence_mbar_init();
  } else if (tid == kAttnThreads - 1) {
    int n = 0;
    for (int b = 0; b < NB; ++b) hslot_s[b] = p.heavy_mask && p.heavy_mask[b] ? (int8_t)n++ : (int8_t)-1;
  }
  if (tid >= kPlanChunks)
    for (int d = tid - kPlanChunks; d < D; d += kAttnThreads - kPlanChunks) perm_s[d] = (int)p.perm[d];
  const int seqs = p.prefix_mode ? 1 : p.B;
  const int rows_total = item_rows_total(p);
  const int mtiles = (rows_total + ROWS - 1) / ROWS;
  const int per = (seqs + kPlanChunks - 1) / kPlanChunks;
  if (tid < kPlanChunks) {
    int n = 0;
    for (int i = tid * per; i < min(seqs, (tid + 1) * per); ++i) {
      const int len = own_length(p, i);
      n += tiles_of(len) + ITEM;
      if (per == 1) len_s[i] = len;
    }
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += u;
    }
    cum_s[tid + 1] = n;          // within the warp's 32 chunks
  }
  if (tid == 0) cum_s[0] = 0;
  __syncthreads();
  int before = 0;
  if (tid < kPlanChunks)
    for (int i = 0; i < warp; ++i) before += cum_s[i * 32 + 32];
  __syncthreads();
  if (tid < kPlanChunks) cum_s[tid + 1] += before;
  __syncthreads();

  // ---- this CTA's range.  With a codebook per head, a head's tiles are followed by kHeadTiles that stand for the
  // change and a range falls into one portion per head; with one codebook for all it is one portion.
  // An item's tiles are followed by ITEM ones that stand for its queries and result.  The entry refuses calls whose
  // tiles may not fit into 31 bits.
  const int per_head = cum_s[kPlanChunks] * mtiles;
  const int gap = p.n_cb > 1 ? kHeadTiles : 0;
  const int stride = per_head + gap, total = stride * p.H - gap;
  const int cta = blockIdx.x;
  const int grid = min((int)gridDim.x, (total + kMinTiles - 1) / kMinTiles);
  asm volatile("griddepcontrol.launch_dependents;");           // the join waits for this grid's end by itself
  // What comes before this grid is done: before the prefix's sets are read, and in every CTA, since what follows this grid
  // counts on that, too.
  auto prefix_written = [&]() {
    if (p.overlap) asm volatile("griddepcontrol.wait;" ::: "memory");
  };
  if (cta >= grid) {
    if (tid == 0) p.desc[cta] = make_int4(0, -1, 0, 0);
    prefix_written();
    return;
  }
  // part i of n of a range of `size`: the first size % n parts are one longer
  auto part = [](int size, int i, int n) { return size / n * i + min(i, size % n); };
  const int from = part(total, cta, grid), to = part(total, cta + 1, grid);
  const int h0 = from / stride, h1 = (to - 1) / stride;
  const int portions = gap ? h1 - h0 + 1 : 1;
  auto length_of = [&](int b) { return per == 1 ? len_s[b] : own_length(p, b); };

  const int pair = warp & (kPairs - 1);
  Walk w;
  // n more tiles of the item are walked: where they end it, on to the next one's first
  auto next_item = [&](int n) {
    w.at += n;
    if (w.t + n < w.tiles) return;               // cut: the range ends here
    w.at += w.tiles + ITEM - (w.t + n);
    w.t = 0;
    if (++w.mt < mtiles) return;
    w.mt = 0;
    if (++w.b == seqs) {
      w.b = 0;
      ++w.h;
    }
    if (w.at < w.end) {
      w.len = length_of(w.b);
      w.tiles = tiles_of(w.len);
    }
  };
  // the pair's part of portion k, in tiles without gaps
  auto enter = [&](int k) {
    int a = from, b = to;
    if (gap) {
      const int h = h0 + k;
      a = max(from - h * stride, 0) + h * per_head;
      b = min(to - h * stride, per_head) + h * per_head;
      a = min(a, b);                           // the range begins in the gap behind head h
    }
    w.at = pair < p.pairs ? a + part(b - a, pair, p.pairs) : b;
    w.end = pair < p.pairs ? a + part(b - a, pair + 1, p.pairs) : b;
    if (w.at >= w.end) return;
    w.h = w.at / per_head;
    int o = w.at - w.h * per_head;
    int lo = 0, hi = kPlanChunks - 1;          // last chunk that begins at or before o
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cum_s[mid] * mtiles <= o) lo = mid;
      else hi = mid - 1;
    }
    o -= cum_s[lo] * mtiles;
    w.b = lo * per;
    w.len = length_of(w.b);
    w.tiles = tiles_of(w.len);
    while (o >= (w.tiles + ITEM) * mtiles) {
      o -= (w.tiles + ITEM) * mtiles;
      ++w.b;
      w.len = length_of(w.b);
      w.tiles = tiles_of(w.len);
    }
    w.mt = o / (w.tiles + ITEM);
    w.t = o - w.mt * (w.tiles + ITEM);
    if (w.t >= w.tiles) next_item(0);
  };
  uint8_t* const my_ring = ring + (size_t)pair * ring_bytes;
  uint64_t* const full = full_s + pair * p.stages;
  uint64_t* const empty = empty_s + pair * p.stages;
  int stage = 0, phase = 0;                    // of the pair's next tile

  if (warp >= kPairs) {
    // ------------------------------------------------------------------ producer
    // Each lane finds the pool row of one of the next 32 copies (and reads the page numbers of the 32 after them
    // ahead); lane 0 then only waits for a stage and issues.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
    const int two = p.chunk != kTile;          // two copies make a tile
    const int vbytes = p.chunk * DV * 2, ibytes = p.chunk * NB, hbytes = p.chunk * p.n_heavy * BD * 2;
    const uint8_t* const heavy = reinterpret_cast<const uint8_t*>(p.heavy);
    const unsigned ps = (unsigned)p.ps;
    for (int k = 0; k < portions; ++k) {
      enter(k);
      while (w.at < w.end) {
        const int n = min(w.end - w.at, w.tiles - w.t);
        const int32_t* table = p.table + (int64_t)w.b * p.table_stride;
        // first token of this lane's copy in the group of tiles from number j on; -1: none
        auto token_of = [&](int j) {
          j += lane >> two;
          const int tok = (w.t + j) * kTile + (two ? (lane & 1) * 16 : 0);
          return j < n && tok < w.len ? tok : -1;
        };
        int tok = token_of(0);
        int ahead = tok >= 0 ? table[(unsigned)tok / ps] : -1;
        if (w.len < 0 && lane == 0) record_error(p.err, kErrLength);
        const int group = 32 >> two;
        for (int j = 0; j < n; j += group) {
          const int page = ahead;
          const bool found = tok >= 0 && page >= 0 && page < p.num_pages;
          if (tok >= 0 && !found) record_error(p.err, kErrPage);
          // -1: no copy, -2: an invalid page
          const int row =
              found ? (int)(((unsigned)page * (unsigned)p.H + (unsigned)w.h) * ps + (unsigned)tok % ps) : (tok >= 0 ? -2 : -1);
          tok = token_of(j + group);
          ahead = tok >= 0 ? table[(unsigned)tok / ps] : -1;
          const int tiles = min(group, n - j);
          for (int i = 0; i < tiles; ++i) {
            const int ra = __shfl_sync(0xffffffffu, row, i << two);
            const int rb = two ? __shfl_sync(0xffffffffu, row, 2 * i + 1) : -1;
            if (lane == 0) {
              mbar_wait(&empty[stage], phase ^ 1, p.err, kErrWait);
              uint8_t* const st = my_ring + stage * p.stage_bytes;
              bad_s[pair * p.stages + stage] = w.len < 0 || ra == -2 || rb == -2;
              mbar_arrive_expect_tx(&full[stage], ((ra >= 0) + (rb >= 0)) * (vbytes + ibytes + hbytes));
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const int r = c ? rb : ra;
                if (r < 0) continue;
#pragma unroll
                for (int x = 0; x < DV / 64; ++x)
                  tma_load_2d(st + x * kTile * 128 + c * 2048, &vmap, x * 64, r, &full[stage]);
                bulk_g2s(st + p.off_idx + c * ibytes, p.idx + (int64_t)r * NB, ibytes, &full[stage]);
                if (hbytes)
                  bulk_g2s(st + p.off_heavy + c * hbytes, heavy + (int64_t)r * p.n_heavy * BD * 2, hbytes, &full[stage]);
              }
            }
            if (++stage == p.stages) {
              stage = 0;
              phase ^= 1;
            }
          }
        }
        next_item(n);
      }
    }
    __syncwarp();
    return;
  }

  // -------------------------------------------------------------------- consumer
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kConsumerRegs));
  const int g = lane >> 2, t = lane & 3;
  const uint32_t image_a = smem_u32(image);
  uint32_t hmask = 0;                          // bit u: unit u of this lane is a dense block
  for (int u = 0; u < UNITS; ++u) hmask |= (uint32_t)(hslot_s[4 * u + t] >= 0) << u;
  const int rot = g & (ROT - 1);
  const uint32_t byte_sel = 0x4440u | t;       // byte t of an index word
  // codebook column of the unit that slot x of a group loads; a group's blocks fill the columns, groups are 32 KB apart
  uint32_t col_a[ROT];
#pragma unroll
  for (int x = 0; x < ROT; ++x) col_a[x] = image_a + (4 * ((x + rot) & (ROT - 1)) + t) * (2 * BD);
  uint32_t v_off[4];                           // this lane's ldmatrix row of 16 tokens x 16 columns, by column group
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int tok = ((lane >> 4) & 1) * 8 + (lane & 7);
    v_off[d] = tok * 128 + (((2 * d + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
  }
  int4 desc = make_int4(0, -1, 0, 0);
  // pieces of this CTA's pairs, [kPairs][2][ROWS] rows: written and read by this CTA, from L2
  float* const pieces = p.pieces + (int64_t)cta * kPairs * 2 * ROWS * RF;

  for (int k = 0; k < portions; ++k) {
    if (tid == 0) {                            // the portion's codebook; no warp reads the last one any more
      if (k) fence_proxy_async_smem();
      const int cb = p.n_cb == 1 ? 0 : (h0 + k) % p.n_cb;
      mbar_arrive_expect_tx(cb_bar, IMAGE);
      bulk_g2s(image, reinterpret_cast<const uint8_t*>(p.image) + (int64_t)cb * IMAGE, IMAGE, cb_bar);
    }
    const float k_scale = p.image_scale[p.n_cb == 1 ? 0 : (h0 + k) % p.n_cb];
    const DenseScale<T> dense_scale(k_scale);
    enter(k);
    int4 head = make_int4(w.at < w.end ? 0 : -1, 0, 0, 0), tail = make_int4(0, 0, 0, 0);
    bool waited = false;

    while (w.at < w.end) {
      const int n = min(w.end - w.at, w.tiles - w.t);
      const int r0 = w.mt * ROWS, nr = min(ROWS, rows_total - r0);
      // Queries as the B operand: this lane's words of row 8c + g, scaled by a power of two into fp16.  A negative
      // scale goes into their sign, so that the factor of a row's scores is not negative and maxima can be taken
      // before it.
      uint32_t qb[NT][KS][2];
      float f[NT][2];
      const bool limited = p.causal && p.L > 1 && !p.prefix_mode;
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        float mx = 0.f;
        T raw[D / 8][2];
        if (8 * c + g < nr) {
          const RowMap at = row_of(p, w.h, w.b, r0 + 8 * c + g);
          const T* src = reinterpret_cast<const T*>(p.q) + at.b * p.qs[0] + at.hq * p.qs[1] + at.l * p.qs[2];
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            const int d = (4 * (i / WORDS) + t) * BD + 2 * (i % WORDS);
            raw[i][0] = src[perm_s[d]];
            raw[i][1] = src[perm_s[d + 1]];
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 8; ++i) raw[i][0] = raw[i][1] = Elem<T>::from_float(0.f);
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          mx = fmaxf(mx, fmaxf(fabsf(Elem<T>::to_float(raw[i][0])), fabsf(Elem<T>::to_float(raw[i][1]))));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // 2^-e with mx in [2^e, 2^(e+1)), within the exponents that have a normal reciprocal; 1 for 0, infinity
        const int e = (__float_as_int(mx) >> 23) - 127;
        const int ec = mx == 0.f || mx == INF ? 0 : max(-126, min(126, e));
        const float sc = copysignf(__int_as_float((127 - ec) << 23), p.scale_log2);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          qb[c][i / 2][i % 2] = pack2<__half>(Elem<T>::to_float(raw[i][0]) * sc, Elem<T>::to_float(raw[i][1]) * sc);
        const float qf = fabsf(p.scale_log2) * __int_as_float((127 + ec) << 23) / k_scale;
        // this lane's columns of S^T are the rows 8c + 2t + j: their factors
#pragma unroll
        for (int j = 0; j < 2; ++j) f[c][j] = __shfl_sync(0xffffffffu, qf, 4 * (2 * t + j));
      }
      const int seen_all = limited ? max(0, w.len - (p.L - 1)) : w.len;
      if (!waited) {
        mbar_wait(cb_bar, k & 1, p.err, kErrWait);
        waited = true;
      }

      float o[NT][DV / 16][4];
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int i = 0; i < DV / 16; ++i) o[c][i][0] = o[c][i][1] = o[c][i][2] = o[c][i][3] = 0.f;
      // m: the largest score before its factor, or one that it exceeds by at most kSlack after it
      float m[NT][2], l[NT][2];
#pragma unroll
      for (int c = 0; c < NT; ++c) m[c][0] = m[c][1] = -INF, l[c][0] = l[c][1] = 0.f;
      bool bad = false;
      for (int i = 0; i < n; ++i) {
        const int first = (w.t + i) * kTile;
        mbar_wait(&full[stage], phase, p.err, kErrWait);
        uint8_t* const st = my_ring + stage * p.stage_bytes;
        const uint32_t st_a = smem_u32(st);
        bad |= bad_s[pair * p.stages + stage] != 0;
        if (first + kTile > w.len) {               // rows behind the end hold anything: zero times it is not zero
          for (int x = max(0, w.len - first) * (DV / 8) + lane; x < kTile * (DV / 8); x += 32) {
            const int tok = x / (DV / 8), c = x % (DV / 8);
            *reinterpret_cast<uint4*>(st + (c >> 3) * (kTile * 128) + tok * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        float s[MT][NT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t kw[2][D / 8];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int tok = mt * 16 + y * 8 + g;
            uint32_t ib[UNITS];
            const uint32_t idx_a = st_a + p.off_idx + tok * NB;
            unrolled<(UNITS + 3) / 4>([&](auto i) {
              lds_words<UNITS >= 4 ? 16 : 8, 16 * decltype(i)::v>(ib + 4 * decltype(i)::v, idx_a);
            });
            // slot u loads unit (u + rot) mod ROT of its group of ROT units
            unrolled<UNITS>([&](auto i) {
              constexpr int u = decltype(i)::v;
              uint32_t word = ib[u];
#pragma unroll
              for (int x = 1; x < ROT; ++x)
                if (rot == x) word = ib[(u & ~(ROT - 1)) | ((u + x) & (ROT - 1))];
              lds_words<2 * BD, (u / ROT) * 32768>(kw[y] + u * WORDS, col_a[u % ROT] + (__byte_perm(word, 0, byte_sel) << 7));
            });
            // put the units back in order: rotate each group by rot
#pragma unroll
            for (int u0 = 0; u0 < UNITS; u0 += ROT)
#pragma unroll
              for (int bit = 1; bit < ROT; bit <<= 1) {
                uint32_t tmp[ROT * WORDS];
#pragma unroll
                for (int x = 0; x < ROT; ++x)
#pragma unroll
                  for (int z = 0; z < WORDS; ++z)
                    tmp[x * WORDS + z] =
                        (rot & bit) ? kw[y][(u0 + ((x - bit) & (ROT - 1))) * WORDS + z] : kw[y][(u0 + x) * WORDS + z];
#pragma unroll
                for (int x = 0; x < ROT * WORDS; ++x) kw[y][u0 * WORDS + x] = tmp[x];
              }
            if (p.n_heavy) {                       // dense blocks take the place of their codeword 0
#pragma unroll
              for (int u = 0; u < UNITS; ++u)
                if ((hmask >> u) & 1) {
                  uint32_t* dst = kw[y] + u * WORDS;
                  lds_words<2 * BD, 0>(dst, st_a + p.off_heavy + (tok * p.n_heavy + hslot_s[4 * u + t]) * (2 * BD));
#pragma unroll
                  for (int x = 0; x < WORDS; ++x) dst[x] = dense_scale(dst[x]);
                }
            }
          }
#pragma unroll
          for (int c = 0; c < NT; ++c) {
            s[mt][c][0] = s[mt][c][1] = s[mt][c][2] = s[mt][c][3] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
              mma_f16(s[mt][c], kw[0][2 * ks], kw[1][2 * ks], kw[0][2 * ks + 1], kw[1][2 * ks + 1], qb[c][ks][0],
                      qb[c][ks][1]);
          }
        }
        // online softmax, in powers of two
        const bool edge = first + kTile > seen_all;
        if (edge) {
#pragma unroll
          for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // tokens that row 8c + 2t + j sees
              const int seen = limited ? max(0, w.len - (p.L - 1 - (r0 + 8 * c + 2 * t + j) % p.L)) : w.len;
#pragma unroll
              for (int e = 0; e < 2 * MT; ++e)
                if (first + e * 8 + g >= seen) s[e >> 1][c][(e & 1) * 2 + j] = -INF;
            }
        }
        bool grows = false;
        float top[NT][2];
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            top[c][j] = fmaxf(fmaxf(s[0][c][j], s[0][c][j + 2]), fmaxf(s[1][c][j], s[1][c][j + 2]));
            grows |= m[c][j] == -INF ? top[c][j] != -INF : (top[c][j] - m[c][j]) * f[c][j] > kSlack;
          }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
          for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float x = top[c][j];
#pragma unroll
              for (int of = 4; of < 32; of <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, of));
              const float nm = fmaxf(m[c][j], x);
              const float e = m[c][j] == -INF ? 0.f : fast_exp2((m[c][j] - nm) * f[c][j]);
              m[c][j] = nm;
              l[c][j] *= e;
#pragma unroll
              for (int d = 0; d < DV / 16; ++d) {
                o[c][d][j] *= e;
                o[c][d][j + 2] *= e;
              }
            }
        }
        uint32_t pb[MT][NT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int c = 0; c < NT; ++c) {
            float e[4];
            const float mb[2] = {m[c][0] == -INF ? 0.f : m[c][0], m[c][1] == -INF ? 0.f : m[c][1]};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              if constexpr (kShift<T> != 0.f) e[x] = fast_exp2(fmaf(s[mt][c][x] - mb[x & 1], f[c][x & 1], kShift<T>));
              else e[x] = fast_exp2((s[mt][c][x] - mb[x & 1]) * f[c][x & 1]);
            }
            if (edge) {                            // -inf times a factor of zero
#pragma unroll
              for (int x = 0; x < 4; ++x) e[x] = s[mt][c][x] == -INF ? 0.f : e[x];
            }
            l[c][0] += e[0] + e[2];
            l[c][1] += e[1] + e[3];
            pb[mt][c][0] = movmatrix(pack2<T>(e[0], e[1]));
            pb[mt][c][1] = movmatrix(pack2<T>(e[2], e[3]));
          }
        unrolled<MT * DV / 16>([&](auto i) {
          constexpr int mt = decltype(i)::v / (DV / 16), d = decltype(i)::v % (DV / 16);
          uint32_t v[4];
          ldmatrix_x4_trans<(d >> 2) * (kTile * 128) + mt * 2048>(v, st_a + v_off[d & 3]);
#pragma unroll
          for (int c = 0; c < NT; ++c) mma_pv<T>(o[c][d], v[0], v[1], v[2], v[3], pb[mt][c][0], pb[mt][c][1]);
        });
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      // the item's or piece's result
      bad = __any_sync(0xffffffffu, bad);
      const bool begins = w.t == 0, ends = w.t + n == w.tiles;
      if (begins && ends) prefix_written();
      uint32_t odd = 0;                            // this lane's rows whose sums are no numbers
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int of = 4; of < 32; of <<= 1) l[c][j] += __shfl_xor_sync(0xffffffffu, l[c][j], of);
          if (bad) l[c][j] = __int_as_float(0x7fffffff);
          else if (l[c][j] != l[c][j]) odd |= 1u << (2 * c + j);
          m[c][j] = m[c][j] == -INF ? -INF : m[c][j] * f[c][j] - kShift<T>;
        }
      for (odd = p.n_heavy ? odd : 0; odd; odd &= odd - 1) {
        const int x = __ffs(odd) - 1, r = 8 * (x >> 1) + 2 * t + (x & 1);
        if (r < nr) report_dense<D, T>(p, row_of(p, w.h, w.b, r0 + r));
      }
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = 8 * c + 2 * t + j;
          float* dst = nullptr;
          if (!(begins && ends)) dst = pieces + ((pair * 2 + begins) * ROWS + r) * RF;
          else if (p.prefix_mode && r < nr) dst = p.prefix_part + flat_row(p, row_of(p, w.h, w.b, r0 + r)) * RF;
          if (dst) {
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) {
              dst[d * 16 + g] = o[c][d][j];
              dst[d * 16 + 8 + g] = o[c][d][j + 2];
            }
            if (g == 0) *reinterpret_cast<float2*>(dst + DV) = make_float2(m[c][j], l[c][j]);
          } else if (begins && ends && r < nr) {
            const int64_t row = flat_row(p, row_of(p, w.h, w.b, r0 + r));
            const Finish e = finish_of<DV>(p, row, m[c][j], l[c][j]);
            T* out = reinterpret_cast<T*>(p.out) + row * DV;
            const int64_t rows = (int64_t)p.B * p.Hq * p.L;
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) {
              o[c][d][j] *= e.f;
              o[c][d][j + 2] *= e.f;
            }
            for (int y = 0; y < p.prefix_parts; ++y) {
              const float* src = p.prefix_part + (y * rows + row) * RF;
              const float fk = fast_exp2(src[DV] - e.base);
#pragma unroll
              for (int d = 0; d < DV / 16; ++d) {
                o[c][d][j] = fmaf(src[d * 16 + g], fk, o[c][d][j]);
                o[c][d][j + 2] = fmaf(src[d * 16 + 8 + g], fk, o[c][d][j + 2]);
              }
            }
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) {
              out[d * 16 + g] = Elem<T>::from_float(o[c][d][j] * e.inv);
              out[d * 16 + 8 + g] = Elem<T>::from_float(o[c][d][j + 2] * e.inv);
            }
          }
        }
      if (!begins) head = make_int4(ends ? 2 : 1, w.h, w.b, w.mt);
      else if (!ends) tail = make_int4(1, w.h, w.b, w.mt);
      next_item(n);
    }
    if (!waited) mbar_wait(cb_bar, k & 1, p.err, kErrWait);      // a pair without tiles: the barrier keeps its phase
    if (lane == 0) {
      head_s[pair] = head;
      tail_s[pair] = tail;
    }
    prefix_written();
    named_barrier(1, kPairs * 32);

    // Items cut between pairs, in the list's order: each starts with a pair's tail piece (or, begun by an earlier
    // CTA, with the first head piece) and goes on through head pieces to the first that ends.  A warp takes one row
    // of one item at a time, all of its pieces in flight at once.
    const int4 hd = lane < kPairs ? head_s[lane] : make_int4(-1, 0, 0, 0);
    const unsigned some = __ballot_sync(0xffffffffu, hd.x >= 0), heads = __ballot_sync(0xffffffffu, hd.x > 0);
    const unsigned last = __ballot_sync(0xffffffffu, hd.x == 2);
    const unsigned tails = __ballot_sync(0xffffffffu, lane < kPairs && tail_s[lane & (kPairs - 1)].x);
    // chain 0: the first head piece; chain 1 + x: pair x's tail
    unsigned chains = tails << 1 | ((some & (0u - some) & heads) != 0);
    int task = warp;                                           // counts (chain, row) from the first chain on
    for (; chains; chains &= chains - 1) {
      const int x = __ffs(chains) - 2;
      const int first = x < 0 ? __ffs(some) - 1 : x;
      const int4 item = x < 0 ? head_s[first] : tail_s[x];
      const unsigned behind = x < 0 ? ~0u << first : ~1u << x;
      const unsigned ends = last & behind;
      const unsigned upto = ends ? (ends & (0u - ends)) * 2 - 1 : ~0u;
      const unsigned members = heads & behind & upto;          // whose head pieces belong to it
      const int nr = min(ROWS, rows_total - item.w * ROWS);
      if (x < 0) desc.x = ends ? 2 : 1;
      else if (!ends) desc = make_int4(desc.x, item.y, item.z, item.w);
      for (; task < nr; task += kPairs) {
        const int d = lane * 4;
        if (d < DV) {
          float m[kPairs + 1], l[kPairs + 1], M = -INF;
          float4 a[kPairs + 1];
#pragma unroll
          for (int z = 0; z <= kPairs; ++z) {
            const bool in = z < kPairs ? (members >> z) & 1 : x >= 0;
            m[z] = -INF;
            if (in) {
              const float* src = pieces + ((z < kPairs ? 2 * z : 2 * x + 1) * ROWS + task) * RF;
              const float2 ml = *reinterpret_cast<const float2*>(src + DV);
              m[z] = ml.x;
              l[z] = ml.y;
              a[z] = *reinterpret_cast<const float4*>(src + d);
            }
          }
#pragma unroll
          for (int z = 0; z <= kPairs; ++z) M = fmaxf(M, m[z]);
          const float base = M == -INF ? 0.f : M;
          float ls = 0.f;
          float4 as = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int i = 0; i <= kPairs; ++i) {
            const int z = (i + kPairs) % (kPairs + 1);         // the tail first
            const bool in = z < kPairs ? (members >> z) & 1 : x >= 0;
            if (in) {
              const float e = fast_exp2(m[z] - base);
              ls = fmaf(l[z], e, ls);
              as = make_float4(fmaf(a[z].x, e, as.x), fmaf(a[z].y, e, as.y), fmaf(a[z].z, e, as.z), fmaf(a[z].w, e, as.w));
            }
          }
          if (x >= 0 && ends) {
            finish4<T, DV>(p, row_of(p, item.y, item.z, item.w * ROWS + task), d, M, ls, as);
          } else {
            float* dst = p.slots + ((int64_t)(2 * cta + (x < 0 ? 0 : 1)) * kItemRows + task) * RF;
            *reinterpret_cast<float4*>(dst + d) = as;
            if (d == 0) *reinterpret_cast<float2*>(dst + DV) = make_float2(M, ls);
          }
        }
      }
      task -= nr;
    }
    if (k + 1 < portions) named_barrier(1, kPairs * 32);
  }
  if (tid == 0) p.desc[cta] = desc;
}

// Joins the pieces of items that were cut between CTAs: block (c, r) takes row r of the item that begins in CTA c's
// range and does not end there, in the order of the ranges.
constexpr int kJoinParts = 4;      // parts of an item's pieces that are joined side by side

template <int DV, typename T>
__global__ void __launch_bounds__(kJoinParts * DV / 4) paged_attention_join(const __grid_constant__ AttnParams p) {
  constexpr int RF = row_floats(DV);
  __shared__ int last_s;
  __shared__ float4 acc_s[kJoinParts][DV / 4];
  __shared__ float2 ml_s[kJoinParts];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x, r = blockIdx.y, part = threadIdx.x / (DV / 4), d = threadIdx.x % (DV / 4) * 4;
  const int4 tail = p.desc[c];
  if (tail.y < 0) return;
  const int row = tail.w * p.item_rows + r;
  if (row >= item_rows_total(p)) return;
  if (threadIdx.x == 0) last_s = gridDim.x;
  __syncthreads();
  for (int k = c + 1; k < gridDim.x && last_s == gridDim.x; k += blockDim.x) {
    __syncthreads();
    if (k + threadIdx.x < gridDim.x && p.desc[k + threadIdx.x].x != 1) atomicMin(&last_s, k + (int)threadIdx.x);
    __syncthreads();
  }
  const int n = min(last_s, (int)gridDim.x - 1) - c + 1;       // pieces: c's tail and the heads behind it
  float m = -__int_as_float(0x7f800000), l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = n * part / kJoinParts; k < n * (part + 1) / kJoinParts; ++k) {
    const float* src = p.slots + ((int64_t)(2 * (c + k) + (k == 0)) * kItemRows + r) * RF;
    join4(m, l, a, src[DV], src[DV + 1], *reinterpret_cast<const float4*>(src + d));
  }
  acc_s[part][d / 4] = a;
  if (d == 0) ml_s[part] = make_float2(m, l);
  __syncthreads();
  if (part) return;
  for (int k = 1; k < kJoinParts; ++k) join4(m, l, a, ml_s[k].x, ml_s[k].y, acc_s[k][d / 4]);
  finish4<T, DV>(p, row_of(p, tail.y, tail.z, row), d, m, l, a);
}

template <int D, int DV, int BD, typename T>
int launch_paged_attention(const AttnParams& p, const CUtensorMap& vmap, int grid, cudaStream_t st) {
  // the split of registers waits forever where the block has fewer than it was planned for
  auto* k = p.item_rows == 8 ? paged_attention_kernel<D, DV, BD, T, 1> : paged_attention_kernel<D, DV, BD, T, 2>;
  static std::atomic<uint64_t> done[2];
  if (!ready_kernel((const void*)k, kSmemMax, kLaunchRegs, done[p.item_rows == 8]))
    return set_last_error(SUNSHAPE_E_CUDA, "the paged attention kernel is not available as it was built.");
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.overlap;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kAttnThreads);
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = st;
  // a kernel of this call reads what the one before it wrote: none follows one that was refused
  if (cudaLaunchKernelEx(&cfg, k, p, vmap) != cudaSuccess) return launch_status("paged attention launch");
  // the join may be scheduled while the main grid drains; it waits for its end before it reads
  cfg.gridDim = dim3(grid, p.item_rows);
  cfg.blockDim = dim3(kJoinParts * DV / 4);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, paged_attention_join<DV, T>, p) != cudaSuccess) return launch_status("paged attention join launch");
  return SUNSHAPE_OK;
}

#define SUNSHAPE_PAGED_INSTANCE(D, DV, BD, T) \
  template int launch_paged_attention<D, DV, BD, T>(const AttnParams&, const CUtensorMap&, int, cudaStream_t);
#define SUNSHAPE_PAGED_INSTANCES(D, T)                                                                          \
  SUNSHAPE_PAGED_INSTANCE(D, 64, 2, T) SUNSHAPE_PAGED_INSTANCE(D, 64, 4, T) SUNSHAPE_PAGED_INSTANCE(D, 64, 8, T) \
  SUNSHAPE_PAGED_INSTANCE(D, 128, 2, T) SUNSHAPE_PAGED_INSTANCE(D, 128, 4, T) SUNSHAPE_PAGED_INSTANCE(D, 128, 8, T)

}  // namespace sunshape
