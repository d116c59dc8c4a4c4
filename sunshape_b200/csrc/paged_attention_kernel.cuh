// The memory-bound kernel of paged attention (few query rows per KV head).
//
// Bound by HBM: a token and KV head cost n_blocks + 2 DV bytes (+ dense blocks).  One producer warp keeps a ring
// of tiles in flight (values by TMA with the 128-byte swizzle, index and dense-block rows by bulk copies, page
// by page); eight consumer warps take tiles in turn, each with its own running softmax, and meet only at the
// end of an item.
//
// Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that the few query rows are the N of the
// MMA (8 or 16 of them) and the 32 tokens fill its M.
// S^T multiplies rebuilt keys that never leave registers: the contraction's order is free, so lane t of a quad takes
// whole codewords of the blocks 4u + t -- one shared-memory load of 2 BD bytes from the head's codebook gives the
// A operand of BD / 4 MMA steps, and Q is laid out to match once per item.  Each block's codewords lie in one
// column of the shared-memory banks, and the tokens that share a load phase walk the columns in rotated order, so
// the random gathers are free of bank conflicts; a barrel of selects puts the registers back in order.
// P^T comes from the accumulators of S^T by a register transpose (movmatrix).
#pragma once

#include <type_traits>

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

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

template <int BYTES>
__device__ __forceinline__ void lds_words(uint32_t* w, uint32_t addr) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
  else if constexpr (BYTES == 8)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}

// dense block words (two 16-bit elements each) into the codebook's fp16 scale
template <typename T>
__device__ __forceinline__ uint32_t dense_word(uint32_t w, float s) {
  float lo, hi;
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = *reinterpret_cast<const __half2*>(&w);
    lo = __low2float(v);
    hi = __high2float(v);
  } else {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  }
  return pack2<__half>(lo * s, hi * s);
}

// A running maximum may fall behind by a factor of 2^kSlack before sums and accumulators are rescaled to a new one;
// weights stay below 2^kSlack, in reach of every type.
constexpr float kSlack = 8.f;

// Where a CTA stands in the list of tiles; the producer and every consumer thread walk it alike.
struct Walk {
  int64_t at, end;       // tiles of the list
  int h, b, mt, t;       // the item and the tile within it
  int len, tiles;        // the sequence's length (-1: invalid) and tiles
};

// NT: groups of eight query rows of an item (1: items have at most eight rows)
template <int D, int DV, int BD, typename T, int NT>
__global__ void __launch_bounds__(kAttnThreads, 1)
    paged_attention_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap vmap) {
  constexpr int NB = D / BD, UNITS = NB / 4, WORDS = BD / 2;   // units: gathers of a lane per token
  constexpr int ROT = 16 / BD;                                 // tokens that share a load phase and a column set
  constexpr int KS = D / 16, ROWS = 8 * NT;
  constexpr int IMAGE = D * 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const ring = base;
  uint8_t* const image = ring + (size_t)p.stages * p.stage_bytes;
  float* const acc_s = reinterpret_cast<float*>(image + IMAGE);              // [consumers][ROWS][DV + 2]
  __half* const q_s = reinterpret_cast<__half*>(acc_s + kConsumers * ROWS * (DV + 2));        // [ROWS][D + 8]
  float* const qf_s = reinterpret_cast<float*>(q_s + ROWS * (D + 8));        // [ROWS] factor of a row's scores
  int* const perm_s = reinterpret_cast<int*>(qf_s + ROWS);                   // [D]
  int64_t* const cum_s = reinterpret_cast<int64_t*>(perm_s + D);             // [kPlanChunks + 1]
  uint64_t* const full = reinterpret_cast<uint64_t*>(cum_s + kPlanChunks + 1);
  uint64_t* const empty = full + p.stages;
  uint64_t* const cb_bar = empty + p.stages;
  // number of the tile that a stage holds or waits for, times 2, plus 1 where its pages are invalid
  volatile int* const tag_s = reinterpret_cast<volatile int*>(cb_bar + 1);   // [stages]
  int8_t* const hslot_s = reinterpret_cast<int8_t*>(cb_bar + 1) + 4 * p.stages;   // [NB] dense slot, -1: codeword
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float INF = __int_as_float(0x7f800000);

  // ---- set-up and plan: prefix sums of tiles over chunks of sequences
  if (tid == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      tag_s[i] = -1;
    }
    mbar_init(cb_bar, 1);
    fence_mbar_init();
    int n = 0;
    for (int b = 0; b < NB; ++b) hslot_s[b] = p.heavy_mask && p.heavy_mask[b] ? (int8_t)n++ : (int8_t)-1;
  }
  for (int d = tid; d < D; d += kAttnThreads) perm_s[d] = (int)p.perm[d];
  const int seqs = p.prefix_mode ? 1 : p.B;
  const int mtiles = (item_rows_total(p) + kItemRows - 1) / kItemRows;
  const int per = (seqs + kPlanChunks - 1) / kPlanChunks;
  if (tid < kPlanChunks) {
    int64_t n = 0;
    for (int i = tid * per; i < min(seqs, (tid + 1) * per); ++i) n += tiles_of(own_length(p, i));
    int64_t v = n;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    cum_s[tid + 1] = v;          // within the warp's 32 chunks
  }
  if (tid == 0) cum_s[0] = 0;
  __syncthreads();
  int64_t before = 0;
  if (tid < kPlanChunks)
    for (int i = 0; i < warp; ++i) before += cum_s[i * 32 + 32];
  __syncthreads();
  if (tid < kPlanChunks) cum_s[tid + 1] += before;
  __syncthreads();
  const int64_t per_head = cum_s[kPlanChunks] * mtiles, total = per_head * p.H;
  const int grid = (int)min((int64_t)gridDim.x, total), cta = blockIdx.x;
  if (cta >= grid) {
    if (tid == 0) p.desc[cta] = make_int4(0, -1, 0, 0);
    return;
  }
  Walk w;
  w.at = total * cta / grid;
  w.end = total * (cta + 1) / grid;
  {
    w.h = (int)(w.at / per_head);
    int64_t o = w.at - w.h * per_head;
    int lo = 0, hi = kPlanChunks - 1;        // last chunk that begins at or before o
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cum_s[mid] * mtiles <= o) lo = mid;
      else hi = mid - 1;
    }
    o -= cum_s[lo] * mtiles;
    w.b = lo * per;
    w.len = own_length(p, w.b);
    w.tiles = tiles_of(w.len);
    while (o >= (int64_t)w.tiles * mtiles) {
      o -= (int64_t)w.tiles * mtiles;
      ++w.b;
      w.len = own_length(p, w.b);
      w.tiles = tiles_of(w.len);
    }
    w.mt = (int)(o / w.tiles);
    w.t = (int)(o - (int64_t)w.mt * w.tiles);
  }
  auto next_item = [&](int n) {              // n: tiles of the item just walked
    w.at += n;
    w.t = 0;
    if (++w.mt < mtiles) return;
    w.mt = 0;
    if (++w.b == seqs) {
      w.b = 0;
      ++w.h;
    }
    if (w.at < w.end) {
      w.len = own_length(p, w.b);
      w.tiles = tiles_of(w.len);
    }
  };

  if (warp >= kConsumers) {
    // ----------------------------------------------------------------- producers
    // Producer x takes the tiles x, x + kProducers, ... of the CTA's list.  Each lane finds the pool row of one of
    // its next 32 copies (and reads the page numbers of the 32 after them ahead); lane 0 then only waits for a
    // stage and issues.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
    const int x = warp - kConsumers;
    int stage = x, phase = 0, turn = 0, tile = x;   // stages: a multiple of the producers, so each has one of its own
    const int two = p.chunk != kTile;          // two copies make a tile
    const int vbytes = p.chunk * DV * 2, ibytes = p.chunk * NB, hbytes = p.chunk * p.n_heavy * BD * 2;
    const uint8_t* const heavy = reinterpret_cast<const uint8_t*>(p.heavy);
    const unsigned ps = (unsigned)p.ps;
    while (w.at < w.end) {
      const int n = (int)min(w.end - w.at, (int64_t)(w.tiles - w.t));
      const int32_t* table = p.table + (int64_t)w.b * p.table_stride;
      const int i0 = (x - turn + kProducers) % kProducers;          // first of the piece's tiles that is this warp's
      const int mine = n > i0 ? (n - i0 + kProducers - 1) / kProducers : 0;
      // first token of this lane's copy in the group of tiles from number j on; -1: none
      auto token_of = [&](int j) {
        j += lane >> two;
        const int tok = (w.t + i0 + j * kProducers) * kTile + (two ? (lane & 1) * 16 : 0);
        return j < mine && tok < w.len ? tok : -1;
      };
      int tok = token_of(0);
      int ahead = tok >= 0 ? table[(unsigned)tok / ps] : -1;
      if (w.len < 0 && lane == 0) record_error(p.err, kErrLength);
      const int group = 32 >> two;
      for (int j = 0; j < mine; j += group) {
        const int page = ahead;
        const bool found = tok >= 0 && page >= 0 && page < p.num_pages;
        if (tok >= 0 && !found) record_error(p.err, kErrPage);
        const int row =
            found ? (int)(((unsigned)page * (unsigned)p.H + (unsigned)w.h) * ps + (unsigned)tok % ps) : (tok >= 0 ? -2 : -1);
        tok = token_of(j + group);
        ahead = tok >= 0 ? table[(unsigned)tok / ps] : -1;
        const int tiles = min(group, mine - j);
        for (int i = 0; i < tiles; ++i) {
          const int ra = __shfl_sync(0xffffffffu, row, i << two);
          const int rb = two ? __shfl_sync(0xffffffffu, row, 2 * i + 1) : -1;
          if (lane == 0) {
            mbar_wait(&empty[stage], phase ^ 1, p.err, kErrWait);
            uint8_t* const st = ring + (size_t)stage * p.stage_bytes;
            tag_s[stage] = 2 * tile + (w.len < 0 || ra == -2 || rb == -2);
            mbar_arrive_expect_tx(&full[stage], ((ra >= 0) + (rb >= 0)) * (vbytes + ibytes + hbytes));
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int r = k ? rb : ra;
              if (r < 0) continue;
#pragma unroll
              for (int c = 0; c < DV / 64; ++c)
                tma_load_2d(st + c * kTile * 128 + k * 2048, &vmap, c * 64, r, &full[stage]);
              bulk_g2s(st + p.off_idx + k * ibytes, p.idx + (int64_t)r * NB, ibytes, &full[stage]);
              if (hbytes)
                bulk_g2s(st + p.off_heavy + k * hbytes, heavy + (int64_t)r * p.n_heavy * BD * 2, hbytes, &full[stage]);
            }
          }
          tile += kProducers;
          stage += kProducers;
          if (stage == p.stages + x) {
            stage = x;
            phase ^= 1;
          }
        }
      }
      turn = (turn + n) % kProducers;
      next_item(n);
    }
    __syncwarp();
    return;
  }

  // -------------------------------------------------------------------- consumers
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kConsumerRegs));
  const int g = lane >> 2, t = lane & 3;
  const uint32_t image_a = smem_u32(image);
  int head = -1, cb_phase = 0;
  float k_scale = 1.f;
  uint32_t hmask = 0;                          // bit u: unit u of this lane is a dense block
  for (int u = 0; u < UNITS; ++u) hmask |= (uint32_t)(hslot_s[4 * u + t] >= 0) << u;
  const int rot = g & (ROT - 1);
  const uint32_t byte_sel = 0x4440u | t;       // byte t of an index word
  uint32_t col_a[UNITS];                       // codebook column of the unit that slot u loads
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int b = 4 * ((u & ~(ROT - 1)) | ((u + rot) & (ROT - 1))) + t;
    col_a[u] = image_a + (b / (64 / BD)) * 32768 + (b % (64 / BD)) * (2 * BD);
  }
  uint32_t v_off[4];                           // this lane's ldmatrix row of 16 tokens x 16 columns, by column group
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int tok = ((lane >> 4) & 1) * 8 + (lane & 7);
    v_off[d] = tok * 128 + (((2 * d + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
  }
  int turn = 0;                                // warp that takes the next tile of the CTA's list
  int stage = warp % p.stages, phase = (warp / p.stages) & 1, tile = warp;   // this warp's next tile
  int head_piece = 0;
  int4 tail = make_int4(0, -1, 0, 0);
  const int rows_total = item_rows_total(p);

  while (w.at < w.end) {
    const int n = (int)min(w.end - w.at, (int64_t)(w.tiles - w.t));
    const int r0 = w.mt * kItemRows, nr = min(kItemRows, rows_total - r0);
    // the head's codebook
    if (w.h != head) {
      const int cb = p.n_cb == 1 ? 0 : w.h % p.n_cb;
      if (head < 0 || p.n_cb > 1) {
        if (tid == 0) {                        // no warp reads the old codebook: the last item's barriers
          fence_proxy_async_smem();
          mbar_arrive_expect_tx(cb_bar, IMAGE);
          bulk_g2s(image, reinterpret_cast<const uint8_t*>(p.image) + (int64_t)cb * IMAGE, IMAGE, cb_bar);
        }
        k_scale = p.image_scale[cb];
      }
    }
    // queries of the item: permuted, scaled by a power of two into fp16; a negative scale goes into their sign, so
    // that the factor of a row's scores is not negative and maxima can be taken before it
    for (int r = warp; r < ROWS; r += kConsumers) {
      float x[D / 32], mx = 0.f;
      if (r < nr) {
        const RowMap at = row_of(p, w.h, w.b, r0 + r);
        const T* src = reinterpret_cast<const T*>(p.q) + at.b * p.qs[0] + at.hq * p.qs[1] + at.l * p.qs[2];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          x[i] = Elem<T>::to_float(src[perm_s[i * 32 + lane]]);
          mx = fmaxf(mx, fabsf(x[i]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) x[i] = 0.f;
      }
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      // 2^-e with mx in [2^e, 2^(e+1)), within the exponents that have a normal reciprocal; 1 for 0, infinity
      const int e = (__float_as_int(mx) >> 23) - 127;
      const int ec = mx == 0.f || mx == INF ? 0 : max(-126, min(126, e));
      const float s = copysignf(__int_as_float((127 - ec) << 23), p.scale_log2);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) q_s[r * (D + 8) + i * 32 + lane] = __float2half_rn(x[i] * s);
      if (lane == 0) qf_s[r] = fabsf(p.scale_log2) * __int_as_float((127 + ec) << 23) / k_scale;
    }
    named_barrier(1, kConsumers * 32);
    if (w.h != head) {
      if (head < 0 || p.n_cb > 1) {
        mbar_wait(cb_bar, cb_phase, p.err, kErrWait);
        cb_phase ^= 1;
      }
      head = w.h;
    }
    uint32_t qb[NT][KS][2];
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int word = 2 * ks + i, u = word / WORDS;
          const int d = (4 * u + t) * BD + 2 * (word % WORDS);
          qb[c][ks][i] = *reinterpret_cast<const uint32_t*>(q_s + (8 * c + g) * (D + 8) + d);
        }
    // this lane's rows are 8c + 2t + j: their score factors, and the tokens that each sees
    const bool limited = p.causal && p.L > 1 && !p.prefix_mode;
    float f[NT][2];
    int seen[NT][2];
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        f[c][j] = qf_s[8 * c + 2 * t + j];
        seen[c][j] = limited ? max(0, w.len - (p.L - 1 - (r0 + 8 * c + 2 * t + j) % p.L)) : w.len;
      }
    const int seen_all = limited ? max(0, w.len - (p.L - 1)) : w.len;

    float o[NT][DV / 16][4];
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int i = 0; i < DV / 16; ++i) o[c][i][0] = o[c][i][1] = o[c][i][2] = o[c][i][3] = 0.f;
    // m: the largest score before its factor, or one that it exceeds by at most kSlack after it; mb: m, 0 for none yet
    float m[NT][2], mb[NT][2], l[NT][2];
#pragma unroll
    for (int c = 0; c < NT; ++c) m[c][0] = m[c][1] = -INF, mb[c][0] = mb[c][1] = l[c][0] = l[c][1] = 0.f;
    bool bad = false;
    const int w0 = turn;                                           // warp of the piece's first tile
    for (int i = (warp - w0 + kConsumers) % kConsumers; i < n; i += kConsumers) {
      const int first = (w.t + i) * kTile;
      // Tiles of a stage go to different warps: only the tag tells that the stage has come to this one, and that its
      // barrier cannot be a whole turn behind, where the wait for a parity would pass at once.
      int tag = tag_s[stage];
      if (tag >> 1 != tile) {
        const uint64_t t0 = global_ns();
        while ((tag = tag_s[stage]) >> 1 != tile)
          if (global_ns() - t0 > kWaitLimitNs) {
            record_error(p.err, kErrWait);
            break;
          }
      }
      mbar_wait(&full[stage], phase, p.err, kErrWait);
      tile += kConsumers;
      uint8_t* const st = ring + (size_t)stage * p.stage_bytes;
      const uint32_t st_a = smem_u32(st);
      bad |= tag & 1;
      float s[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint32_t kw[2][D / 8];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int tok = mt * 16 + y * 8 + g;
          uint32_t ib[UNITS];
#pragma unroll
          for (int u = 0; u < UNITS; u += 4) {
            if constexpr (UNITS >= 4) lds_words<16>(ib + u, st_a + p.off_idx + tok * NB + u * 4);
            else lds_words<8>(ib + u, st_a + p.off_idx + tok * NB + u * 4);
          }
          // slot u loads unit (u + r) mod ROT of its group of ROT units
#pragma unroll
          for (int u = 0; u < UNITS; ++u) {
            uint32_t word = ib[u];
#pragma unroll
            for (int x = 1; x < ROT; ++x)
              if (rot == x) word = ib[(u & ~(ROT - 1)) | ((u + x) & (ROT - 1))];
            lds_words<2 * BD>(kw[y] + u * WORDS, col_a[u] + (__byte_perm(word, 0, byte_sel) << 7));
          }
          // put the units back in order: rotate each group by r
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
                lds_words<2 * BD>(dst, st_a + p.off_heavy + (tok * p.n_heavy + hslot_s[4 * u + t]) * (2 * BD));
#pragma unroll
                for (int x = 0; x < WORDS; ++x) dst[x] = dense_word<T>(dst[x], k_scale);
              }
          }
        }
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          s[mt][c][0] = s[mt][c][1] = s[mt][c][2] = s[mt][c][3] = 0.f;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
            mma_f16(s[mt][c], kw[0][2 * ks], kw[1][2 * ks], kw[0][2 * ks + 1], kw[1][2 * ks + 1], qb[c][ks][0], qb[c][ks][1]);
        }
      }
      // online softmax, in powers of two
      const bool edge = first + kTile > seen_all;
      if (edge) {
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (first + (e >> 2) * 16 + ((e >> 1) & 1) * 8 + g >= seen[c][e & 1]) s[e >> 2][c][e & 3] = -INF;
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
            mb[c][j] = nm == -INF ? 0.f : nm;
            l[c][j] *= e;
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) {
              o[c][d][j] *= e;
              o[c][d][j + 2] *= e;
            }
          }
      }
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          float e[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) e[x] = fast_exp2((s[mt][c][x] - mb[c][x & 1]) * f[c][x & 1]);
          if (edge) {                            // -inf times a factor of zero
#pragma unroll
            for (int x = 0; x < 4; ++x) e[x] = s[mt][c][x] == -INF ? 0.f : e[x];
          }
          l[c][0] += e[0] + e[2];
          l[c][1] += e[1] + e[3];
          pb[mt][c][0] = movmatrix(pack2<T>(e[0], e[1]));
          pb[mt][c][1] = movmatrix(pack2<T>(e[2], e[3]));
        }
      if (first + kTile > w.len) {               // rows behind the end hold anything: zero times it is not zero
        for (int k = max(0, w.len - first) * (DV / 8) + lane; k < kTile * (DV / 8); k += 32) {
          const int tok = k / (DV / 8), c = k % (DV / 8);
          *reinterpret_cast<uint4*>(st + (c >> 3) * (kTile * 128) + tok * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int d = 0; d < DV / 16; ++d) {
          uint32_t v[4];
          ldmatrix_x4_trans(v, st_a + v_off[d & 3] + (d >> 2) * (kTile * 128) + mt * 2048);
#pragma unroll
          for (int c = 0; c < NT; ++c) mma_pv<T>(o[c][d], v[0], v[1], v[2], v[3], pb[mt][c][0], pb[mt][c][1]);
        }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
      stage += kConsumers;                                          // this warp's next tile
      while (stage >= p.stages) {
        stage -= p.stages;
        phase ^= 1;
      }
    }
    turn = (turn + n) % kConsumers;

    // join the warps that took tiles of this piece
    const int warps = min(kConsumers, n);
    const int mine = (warp - w0 + kConsumers) % kConsumers;         // rank among them
    if (mine < warps) {
      bad = __any_sync(0xffffffffu, bad);
      float* dst = acc_s + (size_t)mine * ROWS * (DV + 2);
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int of = 4; of < 32; of <<= 1) l[c][j] += __shfl_xor_sync(0xffffffffu, l[c][j], of);
          float* to = dst + (8 * c + 2 * t + j) * (DV + 2);
          if (g == 0) {
            to[DV] = m[c][j] == -INF ? -INF : m[c][j] * f[c][j];
            to[DV + 1] = bad ? __int_as_float(0x7fffffff) : l[c][j];
          }
#pragma unroll
          for (int d = 0; d < DV / 16; ++d) {
            to[d * 16 + g] = o[c][d][j];
            to[d * 16 + 8 + g] = o[c][d][j + 2];
          }
        }
    }
    named_barrier(1, kConsumers * 32);
    const bool begins = w.t == 0, ends = w.t + n == w.tiles;
    float* slot = begins && ends ? nullptr : p.slots + (int64_t)(2 * cta + (begins ? 1 : 0)) * kItemRows * (DV + 2);
    for (int e = tid; e < nr * DV; e += kConsumers * 32) {
      const int r = e / DV, d = e % DV;
      float M = -INF;
      for (int k = 0; k < warps; ++k) M = fmaxf(M, acc_s[((size_t)k * ROWS + r) * (DV + 2) + DV]);
      const float bs = M == -INF ? 0.f : M;
      float l = 0.f, a = 0.f;
      for (int k = 0; k < warps; ++k) {
        const float* src = acc_s + ((size_t)k * ROWS + r) * (DV + 2);
        const float e = fast_exp2(src[DV] - bs);
        l = fmaf(src[DV + 1], e, l);
        a = fmaf(src[d], e, a);
      }
      if (slot) {
        slot[r * (DV + 2) + 2 + d] = a;
        if (d == 0) {
          slot[r * (DV + 2)] = M;
          slot[r * (DV + 2) + 1] = l;
        }
      } else {
        finish_element<T, DV>(p, row_of(p, w.h, w.b, r0 + r), d, M, l, a);
      }
    }
    if (!begins) head_piece = ends ? 2 : 1;
    else if (!ends) tail = make_int4(0, w.h, w.b, w.mt);
    next_item(n);
  }
  if (tid == 0) {
    tail.x = head_piece;
    p.desc[cta] = tail;
  }
}

// Joins the pieces of items that were cut: block (c, r) takes row r of the item that begins in CTA c's range
// and does not end there, in the order of the ranges.
template <int DV, typename T>
__global__ void __launch_bounds__(DV) paged_attention_join(const __grid_constant__ AttnParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x, r = blockIdx.y, d = threadIdx.x;
  const int4 tail = p.desc[c];
  if (tail.y < 0) return;
  const int row = tail.w * kItemRows + r;
  if (row >= item_rows_total(p)) return;
  int last = c + 1;
  while (last < gridDim.x && p.desc[last].x == 1) ++last;
  const float INF = __int_as_float(0x7f800000);
  const float* own = p.slots + ((int64_t)(2 * c + 1) * kItemRows + r) * (DV + 2);
  float m = own[0], l = own[1], a = own[2 + d];
  for (int k = c + 1; k <= last && k < gridDim.x; ++k) {
    const float* src = p.slots + ((int64_t)(2 * k) * kItemRows + r) * (DV + 2);
    const float mk = src[0], M = fmaxf(m, mk), bs = M == -INF ? 0.f : M;
    const float f = fast_exp2(m - bs), fk = fast_exp2(mk - bs);
    l = l * f + src[1] * fk;
    a = a * f + src[2 + d] * fk;
    m = M;
  }
  finish_element<T, DV>(p, row_of(p, tail.y, tail.z, row), d, m, l, a);
}

template <int D, int DV, int BD, typename T>
int launch_paged_attention(const AttnParams& p, const CUtensorMap& vmap, int grid, cudaStream_t st) {
  // the split of registers waits forever where the block has fewer than it was planned for
  auto* k = p.item_rows == 8 ? paged_attention_kernel<D, DV, BD, T, 1> : paged_attention_kernel<D, DV, BD, T, 2>;
  cudaFuncAttributes fa;
  if (cudaFuncGetAttributes(&fa, k) != cudaSuccess || fa.numRegs != kLaunchRegs)
    return set_last_error(SUNSHAPE_E_CUDA, "paged attention kernel was built for another register count.");
  cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, p.smem);
  k<<<grid, kAttnThreads, p.smem, st>>>(p, vmap);
  // the join may be scheduled while the main grid drains; it waits for its end before it reads
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid, kItemRows);
  cfg.blockDim = dim3(DV);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, paged_attention_join<DV, T>, p);
  return SUNSHAPE_OK;
}

#define SUNSHAPE_PAGED_INSTANCE(D, DV, BD, T) \
  template int launch_paged_attention<D, DV, BD, T>(const AttnParams&, const CUtensorMap&, int, cudaStream_t);
#define SUNSHAPE_PAGED_INSTANCES(D, T)                                                                          \
  SUNSHAPE_PAGED_INSTANCE(D, 64, 2, T) SUNSHAPE_PAGED_INSTANCE(D, 64, 4, T) SUNSHAPE_PAGED_INSTANCE(D, 64, 8, T) \
  SUNSHAPE_PAGED_INSTANCE(D, 128, 2, T) SUNSHAPE_PAGED_INSTANCE(D, 128, 4, T) SUNSHAPE_PAGED_INSTANCE(D, 128, 8, T)

}  // namespace sunshape
