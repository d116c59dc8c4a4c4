// Attention of many query rows over the shared prefix, on the 5th-generation tensor cores.
//
// All sequences' query rows of a KV head attend to the same keys, so a key is rebuilt once for 256 rows and the work is
// two matrix products a tile, S = Q K^T and O += P V (128 rows x 128 tokens x D, and x DV):
//   * one warp copies value tiles by TMA (128-byte swizzle), page by page, two tiles ahead;
//   * four warps rebuild the tile's keys as fp16, one thread a token: its index row lies in a register, read a tile
//     ahead; its codewords come from the head's codebook in shared memory and go, swizzled, into the K operand.  Lanes
//     take the blocks in the order s xor (2 l in GF(8)), for which both the codebook's columns and the swizzled places
//     of eight lanes are all different: neither side has bank conflicts;
//   * one thread issues the tcgen05.mma of both groups of 128 rows in turn -- PV of one group and QK of its next tile
//     while the other group's softmax runs -- with accumulators in tensor memory, S and O of both groups: 512 columns;
//   * eight warps a row group, two threads a row with 64 columns each: scores from tensor memory, weights in powers of
//     two against a maximum that may fall behind by 2^kSlack (then, and only then, O is rescaled in place), P as 16-bit
//     pairs over S.  One thread a row takes about 2150 cycles a tile, during which its group's next products wait.
// Bound: (D + DV) 256 multiply-adds a token and head against one exponential for each row: at D = DV = 128 the tensor
// cores and the special function units both need 2048 cycles a tile of 256 rows, so the two groups' phases must overlap.
// Measured on B200: 512 rows of 8 heads over 32768 tokens (69 GFLOP): 2.5 us a tile of 256 rows, 88 us the kernel with 12 us
// of start and 5 us of results; the whole call, with the sequences' own 180k tokens, 139 us (memory-bound kernel alone: 477).
//
// The list of tiles (head, 256 rows, 128 tokens) is cut into equal ranges as in the memory-bound kernel; pieces of an
// item cut between CTAs go to slots that paged_prefix_join adds up in order.
#pragma once

#include "paged_attention_kernel.cuh"

namespace sunshape {

constexpr int kPfTokens = 128, kPfRows = 256;
// tiles that an item's queries, codebook and result are charged in the split (512 rows over 32768 tokens of 8 heads: 137 us
// with none, 122 with 7, 121 with 14)
constexpr int kPfItemTiles = 14;
constexpr int kPfThreads = 768;    // warps 0: values, 1: MMA, 2-3: none, 4-7: keys, 8-15 and 16-23: softmax of the row groups
constexpr int kPfLaunchRegs = 80, kPfRegs0 = 40, kPfRegsKeys = 88, kPfRegsSoftmax = 88;
static_assert(kPfRegs0 <= kPfLaunchRegs && kPfRegsKeys >= kPfLaunchRegs && kPfRegsSoftmax >= kPfLaunchRegs, "dec and inc");
static_assert(kPfRegs0 + kPfRegsKeys + 4 * kPfRegsSoftmax <= 6 * kPfLaunchRegs, "the split waits forever where it exceeds the launch");

struct PrefixSmem {
  // all operands 1024-byte aligned
  static __host__ __device__ constexpr int q(int d) { return kPfRows * d * 2; }
  static __host__ __device__ constexpr int k(int d) { return kPfTokens * d * 2; }
  static __host__ __device__ constexpr int v(int dv) { return kPfTokens * dv * 2; }
  static __host__ __device__ constexpr int total(int d, int dv) {
    return q(d) + k(d) + 2 * v(dv) + d * 512 + 2 * kPfRows * 4 + 128 + 128;
  }
};

__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo) {
  // start, leading and stride (one 8-row atom) offsets in 16 bytes, version 1, 128-byte swizzle
  return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// kind::f16, fp32 accumulator, M 128, N n; A K-major, B K-major or (mn) with its N contiguous
__host__ __device__ constexpr uint32_t f16_idesc(bool bf16, int n, bool mn) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ void pf_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void pf_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pf_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

#define SUNSHAPE_TM32(OP, PRE, POST)                                                                                       \
  asm volatile("tcgen05." OP ".sync.aligned.32x32b.x32.b32 " PRE                                                            \
               "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28," \
               "%29,%30,%31}" POST ";"

// 32 columns of this warp's lanes
__device__ __forceinline__ void tm_load32(float (&v)[32], uint32_t addr) {
  SUNSHAPE_TM32("ld", "", ", [%32]")
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
                 "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
                 "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
                 "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
               : "r"(addr));
}
// completes the loads before it; v is tied so that no use moves above
__device__ __forceinline__ void tm_wait_load(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(v[i])::"memory");
}
template <typename U>
__device__ __forceinline__ void tm_store32(uint32_t addr, const U* v) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(v);
  SUNSHAPE_TM32("st", "[%32], ", "")::"r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]),
      "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]),
      "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]),
      "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31]), "r"(addr)
      : "memory");
}
// pairs of fp32 numbers in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(r)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(r)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return r;
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<uint64_t&>(r)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return r;
}

__device__ __forceinline__ void tm_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 64 scores of a row to weights 2^((s - mb) f + kShift), as 16-bit pairs, with their sum and the largest score.  Scores from
// `valid` on are left out.
template <typename T, bool TAIL>
__device__ __forceinline__ void tile_weights(uint32_t s_t, int valid, float mb, float f, uint32_t* pk, float& top, float& sum) {
  const float INF = __int_as_float(0x7f800000);
  float t0 = -INF, t1 = -INF;
  float2 acc = make_float2(0.f, 0.f);
  const float2 nb = make_float2(-mb, -mb), ff = make_float2(f, f);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float v[32];
    tm_load32(v, s_t + c * 32);
    tm_wait_load(v);
    if constexpr (TAIL) {
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (c * 32 + e >= valid) v[e] = -INF;
    }
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
      t0 = fmaxf(t0, fmaxf(v[e], v[e + 1]));
      t1 = fmaxf(t1, fmaxf(v[e + 2], v[e + 3]));
    }
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      const float2 d = add2(make_float2(v[e], v[e + 1]), nb);
      float2 y;
      if constexpr (kShift<T> != 0.f) y = fma2(d, ff, make_float2(kShift<T>, kShift<T>));
      else y = mul2(d, ff);
      float2 w = make_float2(fast_exp2(y.x), fast_exp2(y.y));
      if constexpr (TAIL) {             // -inf times a factor of zero
        w.x = c * 32 + e < valid ? w.x : 0.f;
        w.y = c * 32 + e + 1 < valid ? w.y : 0.f;
      }
      acc = add2(acc, w);
      pk[c * 16 + e / 2] = pack2<T>(w.x, w.y);
    }
  }
  top = fmaxf(t0, t1);
  sum = acc.x + acc.y;
}
template <typename T>
__device__ __forceinline__ void tile_weights(uint32_t s_t, int valid, float mb, float f, uint32_t* pk, float& top, float& sum) {
  if (valid < kPfTokens / 2) tile_weights<T, true>(s_t, valid, mb, f, pk, top, sum);
  else tile_weights<T, false>(s_t, valid, mb, f, pk, top, sum);
}

template <int D, int DV, int BD, typename T>
__global__ void __launch_bounds__(kPfThreads, 1)
    paged_prefix_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap vmap) {
  constexpr int NB = D / BD, KS = D / 16, IMAGE = D * 512, RF = row_floats(DV);
  constexpr int HALF = kPfTokens * 128;          // an operand's 64 columns of 128 rows
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) uint8_t q_s[];   // the operands' swizzle counts on the base's alignment
  uint8_t* const k_s = q_s + PrefixSmem::q(D);   // q: [2 groups][D / 64][128 rows][128 bytes], swizzled
  uint8_t* const v_s = k_s + PrefixSmem::k(D);   // [2][DV / 64][128 tokens][128 bytes]
  uint8_t* const image = v_s + 2 * PrefixSmem::v(DV);
  // [2 groups][2 halves][128]: what the two threads of a row tell each other; first, in half 0, the rows' score factors
  float* const row_s = reinterpret_cast<float*>(image + IMAGE);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(row_s + 2 * kPfRows);
  uint64_t *const v_full = bars, *const v_free = bars + 2, *const k_ready = bars + 4, *const k_free = bars + 5,
                  *const s_full = bars + 6, *const p_ready = bars + 8, *const pv_done = bars + 10, *const cb_bar = bars + 12,
                  *const q_ready = bars + 14;
  uint32_t* const tmem_s = reinterpret_cast<uint32_t*>(bars + 13);
  volatile int* const bad_s = reinterpret_cast<volatile int*>(tmem_s + 1);
  int8_t* const hslot_s = reinterpret_cast<int8_t*>(bars + 16);            // [NB] dense slot, -1: codeword
  int8_t* const hblock_s = hslot_s + NB;                                   // [NB] block of a dense slot
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float INF = __int_as_float(0x7f800000);

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_free[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 256);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(k_ready, 128);
    mbar_init(k_free, 1);
    mbar_init(cb_bar, 1);
    mbar_init(q_ready, 512);
    fence_mbar_init();
    *bad_s = 0;
    int n = 0;
    for (int b = 0; b < NB; ++b) {
      const bool dense = p.heavy_mask && p.heavy_mask[b];
      if (dense) hblock_s[n] = (int8_t)b;
      hslot_s[b] = dense ? (int8_t)n++ : (int8_t)-1;
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_s)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    pf_fence_before();
  }
  __syncthreads();
  pf_fence_after();
  asm volatile("griddepcontrol.launch_dependents;");
  const uint32_t tmem = *tmem_s;                 // columns: S0, S1 (128 each), O0, O1 (DV each); P over S

  // this CTA's range of the list (head, group of 256 rows, tile)
  const int rows_total = p.B * p.G * p.L, items = (rows_total + kPfRows - 1) / kPfRows;
  const int tiles = (p.prefix_len + kPfTokens - 1) / kPfTokens;
  // an item's tiles are followed by kPfItemTiles that stand for the rest of its work
  const int stride = tiles + kPfItemTiles, total = stride * items * p.H - kPfItemTiles;
  const int grid = min((int)gridDim.x, total), cta = blockIdx.x;
  auto part = [](int size, int i, int n) { return size / n * i + min(i, size % n); };
  int at = cta < grid ? part(total, cta, grid) : 0;
  const int end = cta < grid ? part(total, cta + 1, grid) : 0;

  // Every role walks the same pieces (a range's part of one item) and meets the others after each: only then are queries
  // and codebook replaced.  it: tiles so far, it1: those of row group 1, which a head's last rows may not
  // fill -- the parities of the barriers.
  int it = 0, it1 = 0, pieces = 0, cb_loads = 0, head = -1;
  int h, t0, n, r0, groups, cb;
  bool load_cb, begins, ends;
  auto next_piece = [&]() {
    int item = at / stride;
    t0 = at - item * stride;
    if (t0 >= tiles) {
      at = ++item * stride;
      t0 = 0;
    }
    if (at >= end) return false;
    n = min(end - at, tiles - t0);
    h = item / items;
    r0 = (item - h * items) * kPfRows;
    groups = rows_total - r0 > 128 ? 2 : 1;
    cb = p.n_cb == 1 ? 0 : h % p.n_cb;
    load_cb = head < 0 || (h != head && p.n_cb > 1);
    cb_loads += load_cb;
    head = h;
    begins = t0 == 0;
    ends = t0 + n == tiles;
    return true;
  };
  auto end_piece = [&]() {
    at += ends ? n + kPfItemTiles : n;
    it += n;
    if (groups == 2) it1 += n;
    ++pieces;
    named_barrier(1, kPfThreads);
    pf_fence_after();
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPfRegs0));
    while (next_piece()) {
      if (load_cb && tid == 0) {
        fence_proxy_async_smem();
        mbar_arrive_expect_tx(cb_bar, IMAGE);
        bulk_g2s(image, reinterpret_cast<const uint8_t*>(p.image) + (int64_t)cb * IMAGE, IMAGE, cb_bar);
      }
      if (warp == 0) {
        // ------------------------------------------------------------------ values
        const unsigned ps = (unsigned)p.ps;
        const int copies = kPfTokens / p.chunk;     // of a tile: 4 or 8
        const int vbytes = p.chunk * DV * 2;
        for (int i = 0; i < n; ++i) {
          const int slot = (it + i) & 1, phase = ((it + i) >> 1) & 1;
          const int tok = (t0 + i) * kPfTokens + lane * p.chunk;
          int row = -1;
          if (lane < copies && tok < p.prefix_len) {
            const int page = p.table[(unsigned)tok / ps];
            if (page >= 0 && page < p.num_pages)
              row = (int)(((unsigned)page * (unsigned)p.H + (unsigned)h) * ps + (unsigned)tok % ps);
            else {
              record_error(p.err, kErrPage);
              *bad_s = 1;
            }
          }
          const unsigned have = __ballot_sync(0xffffffffu, row >= 0);
          if (lane == 0) {
            mbar_wait(&v_free[slot], phase ^ 1, p.err, kErrWait);
            mbar_arrive_expect_tx(&v_full[slot], __popc(have) * vbytes);
          }
          __syncwarp();
          if (row >= 0) {
#pragma unroll
            for (int c = 0; c < DV / 64; ++c)
              tma_load_2d(v_s + slot * PrefixSmem::v(DV) + c * HALF + lane * p.chunk * 128, &vmap, c * 64, row, &v_full[slot]);
          }
          __syncwarp();
        }
      } else if (warp == 1) {
        // --------------------------------------------------------------------- MMA
        if (lane == 0) {
          const uint32_t id_qk = f16_idesc(false, kPfTokens, false), id_pv = f16_idesc(BF16, DV, true);
          const uint64_t qd = smem_desc(smem_u32(q_s), 16), kd = smem_desc(smem_u32(k_s), 16);
          auto qk = [&](int g) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              const uint64_t off = (ks >> 2) * (HALF >> 4) + (ks & 3) * 2;
              tc_mma_ss(tmem + g * 128, qd + g * ((128 * D * 2) >> 4) + off, kd + off, id_qk, ks > 0);
            }
            pf_commit(&s_full[g]);
          };
          auto pv = [&](int g, int i) {
            const uint64_t vd = smem_desc(smem_u32(v_s + ((it + i) & 1) * PrefixSmem::v(DV)), HALF);
#pragma unroll
            for (int ks = 0; ks < kPfTokens / 16; ++ks)
              tc_mma_ts(tmem + 256 + g * DV, tmem + g * 128 + ks * 8, vd + ks * (2048 >> 4), id_pv, i > 0 || ks > 0);
            pf_commit(&pv_done[g]);
          };
          mbar_wait(q_ready, pieces & 1, p.err, kErrWait);
          mbar_wait(k_ready, it & 1, p.err, kErrWait);
          pf_fence_after();
          for (int g = 0; g < groups; ++g) qk(g);
          pf_commit(k_free);
          for (int i = 0; i < n; ++i) {
#pragma unroll 1
            for (int g = 0; g < groups; ++g) {
              mbar_wait(&p_ready[g], (g ? it1 + i : it + i) & 1, p.err, kErrWait);
              if (g == 0) mbar_wait(&v_full[(it + i) & 1], ((it + i) >> 1) & 1, p.err, kErrWait);
              pf_fence_after();
              pv(g, i);
              if (g == groups - 1) pf_commit(&v_free[(it + i) & 1]);
              if (i + 1 < n) {
                if (g == 0) mbar_wait(k_ready, (it + i + 1) & 1, p.err, kErrWait);
                pf_fence_after();
                qk(g);
                if (g == groups - 1) pf_commit(k_free);
              }
            }
          }
        }
        __syncwarp();
      }
      end_piece();
    }
    if (warp == 1) {
      __syncwarp();
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
  } else if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPfRegsKeys));
    while (next_piece()) {
      // -------------------------------------------------------------------- keys
      const int tok_l = tid - 128;               // this thread's token of a tile
      const unsigned ps = (unsigned)p.ps;
      const int l8 = lane & 7, mul = ((l8 << 1) ^ (l8 & 4 ? 0xb : 0)) & 7;   // 2 l in GF(8) modulo x^3 + x + 1
      if (load_cb) mbar_wait(cb_bar, (cb_loads - 1) & 1, p.err, kErrWait);
      const DenseScale<T> dense_scale(p.image_scale[cb]);
      const uint32_t image_a = smem_u32(image);
      uint32_t ib[NB / 4];
      // block_dim 8: a dense block is one 16-byte chunk; a token's first four are read ahead, too
      constexpr int AHEAD = BD == 8 ? 4 : 0;
      uint4 dense_ahead[AHEAD + 1];
      int64_t row = -1;
      auto fetch = [&](int i) {                  // pool row and index row of tile i's token; zeros where there is none
        const int tok = (t0 + i) * kPfTokens + tok_l;
        row = -1;
        if (i < n && tok < p.prefix_len) {
          const int page = p.table[(unsigned)tok / ps];
          if (page >= 0 && page < p.num_pages) row = ((int64_t)page * p.H + h) * ps + (unsigned)tok % ps;
        }
#pragma unroll
        for (int x = 0; x < NB / 4; ++x) ib[x] = 0;
        if (row >= 0) {
          const uint8_t* src = p.idx + row * NB;
          if constexpr (NB == 8) {
            *reinterpret_cast<uint2*>(ib) = *reinterpret_cast<const uint2*>(src);
          } else {
#pragma unroll
            for (int x = 0; x < NB / 16; ++x) reinterpret_cast<uint4*>(ib)[x] = reinterpret_cast<const uint4*>(src)[x];
          }
#pragma unroll
          for (int x = 0; x < AHEAD; ++x)
            if (x < p.n_heavy) dense_ahead[x] = reinterpret_cast<const uint4*>(p.heavy)[row * p.n_heavy + x];
        }
      };
      fetch(0);
      for (int i = 0; i < n; ++i) {
        mbar_wait(k_free, (it + i + 1) & 1, p.err, kErrWait);
        uint8_t* const dst = k_s + tok_l * 128;
        // 16-byte chunk j of each 64-column half: 8 / BD codewords
        constexpr int PER = 8 / BD, WORDS = BD / 2;
#pragma unroll
        for (int half = 0; half < D / 64; ++half) {
          uint32_t chunk[8][4];                  // all loads before the stores, which the compiler can not tell apart
#pragma unroll
          for (int s = 0; s < 8; ++s) {
            const int j = s ^ mul;               // chunk of the half; its blocks are half * 8 * PER + j * PER + x
            uint32_t* const w = chunk[s];
            if constexpr (PER == 1) {
              const uint32_t c = __byte_perm(ib[half * 2], ib[half * 2 + 1], j) & 0xffu;
              lds_words<16, 0>(w, image_a + half * 32768 + (c << 7) + j * 16);
            } else if constexpr (PER == 2) {
              // bytes 2j, 2j + 1 of the half's 16
              const uint32_t word = j < 4 ? (j < 2 ? ib[half * 4] : ib[half * 4 + 1]) : (j < 6 ? ib[half * 4 + 2] : ib[half * 4 + 3]);
              const uint32_t two = word >> (16 * (j & 1));
              lds_words<8, 0>(w, image_a + half * 32768 + ((two & 0xffu) << 7) + j * 16);
              lds_words<8, 0>(w + 2, image_a + half * 32768 + (((two >> 8) & 0xffu) << 7) + j * 16 + 8);
            } else {
              uint32_t word = ib[half * 8];
#pragma unroll
              for (int x = 1; x < 8; ++x)
                if (j == x) word = ib[half * 8 + x];
#pragma unroll
              for (int x = 0; x < 4; ++x)
                lds_words<4, 0>(w + x, image_a + half * 32768 + (((word >> (8 * x)) & 0xffu) << 7) + j * 16 + 4 * x);
            }
          }
#pragma unroll
          for (int s = 0; s < 8; ++s) {
            const int j = s ^ mul;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(dst) + half * HALF + ((j ^ (tok_l & 7)) << 4)),
                         "r"(chunk[s][0]), "r"(chunk[s][1]), "r"(chunk[s][2]), "r"(chunk[s][3])
                         : "memory");
          }
        }
        if (p.n_heavy && row >= 0) {             // dense blocks take the place of their codeword 0
          const T* dense = reinterpret_cast<const T*>(p.heavy) + row * p.n_heavy * BD;
          if constexpr (BD == 8) {
#pragma unroll
            for (int x = 0; x < NB; ++x) {
              if (x >= p.n_heavy) break;
              uint4 w = x < AHEAD ? dense_ahead[x < AHEAD ? x : 0] : reinterpret_cast<const uint4*>(dense)[x];
              w = make_uint4(dense_scale(w.x), dense_scale(w.y), dense_scale(w.z), dense_scale(w.w));
              const int b = hblock_s[x];
              *reinterpret_cast<uint4*>(dst + (b >> 3) * HALF + (((b & 7) ^ (tok_l & 7)) << 4)) = w;
            }
          }
#pragma unroll 4
          for (int b = 0; b < (BD == 8 ? 0 : NB); ++b) {
            const int at_b = hslot_s[b];
            if (at_b < 0) continue;
            uint32_t w[WORDS];
#pragma unroll
            for (int x = 0; x < WORDS; ++x) w[x] = dense_scale(reinterpret_cast<const uint32_t*>(dense + at_b * BD)[x]);
            const int byte = b * BD * 2, j = (byte >> 4) & 7;
            uint8_t* to = dst + (byte >> 7) * HALF + ((j ^ (tok_l & 7)) << 4) + (byte & 15);
#pragma unroll
            for (int x = 0; x < WORDS; ++x) reinterpret_cast<uint32_t*>(to)[x] = w[x];
          }
        }
        const int first = (t0 + i) * kPfTokens;
        fetch(i + 1);
        if (first + kPfTokens > p.prefix_len) {  // rows behind the end hold anything: zero times it is not zero
          mbar_wait(&v_full[(it + i) & 1], ((it + i) >> 1) & 1, p.err, kErrWait);
          if (first + tok_l >= p.prefix_len) {
            uint8_t* vr = v_s + ((it + i) & 1) * PrefixSmem::v(DV) + tok_l * 128;
#pragma unroll
            for (int c = 0; c < DV / 8; ++c) *reinterpret_cast<uint4*>(vr + (c >> 3) * HALF + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(k_ready);
      }
      end_piece();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPfRegsSoftmax));
    while (next_piece()) {
      {
        // queries: 16-byte chunks of permuted elements, 16 (or 8) lanes a row, scaled by a power of two into fp16, a
        // negative scale in their sign
        constexpr int CH = D / 8, RPW = 32 / CH;
        const int c = lane % CH;
        int src_d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) src_d[i] = (int)p.perm[c * 8 + i];
        const float k_scale = p.image_scale[cb];
#pragma unroll 4
        for (int r = (warp - 8) * RPW + lane / CH; r < groups * 128; r += 16 * RPW) {
          float x[8], mx = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = 0.f;
          if (r0 + r < rows_total) {
            const RowMap m = row_of(p, h, 0, r0 + r);
            const T* src = reinterpret_cast<const T*>(p.q) + m.b * p.qs[0] + m.hq * p.qs[1] + m.l * p.qs[2];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = Elem<T>::to_float(src[src_d[i]]);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(x[i]));
#pragma unroll
          for (int o = 1; o < CH; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          const int e = (__float_as_int(mx) >> 23) - 127;
          const int ec = mx == 0.f || mx == INF ? 0 : max(-126, min(126, e));
          const float sc = copysignf(__int_as_float((127 - ec) << 23), p.scale_log2);
          uint4 w;
          w.x = pack2<__half>(x[0] * sc, x[1] * sc);
          w.y = pack2<__half>(x[2] * sc, x[3] * sc);
          w.z = pack2<__half>(x[4] * sc, x[5] * sc);
          w.w = pack2<__half>(x[6] * sc, x[7] * sc);
          const int row = r & 127;
          *reinterpret_cast<uint4*>(q_s + (r >> 7) * (128 * D * 2) + (c >> 3) * HALF + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = w;
          if (c == 0) row_s[(r >> 7) * 256 + (r & 127)] = fabsf(p.scale_log2) * __int_as_float((127 + ec) << 23) / k_scale;
        }
        fence_proxy_async_smem();
      }
      mbar_arrive(q_ready);
      named_barrier(10, 512);                    // the rows' factors
      const int g = (warp - 8) / 8;
      if (g < groups) {
        // ----------------------------------------------------------------- softmax
        const int half = ((warp - 8) >> 2) & 1, rl = (warp & 3) * 32 + lane, r = g * 128 + rl;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_t = tmem + g * 128 + lanes + half * 64, p_t = tmem + g * 128 + lanes + half * 32;
        const uint32_t o_t = tmem + 256 + g * DV + lanes + half * (DV / 2);
        float* const mine = row_s + g * 256 + half * 128 + rl;
        const float* const other = row_s + g * 256 + (half ^ 1) * 128 + rl;
        const int base = g ? it1 : it;
        const int pair_bar = 2 + g * 4 + (warp & 3);   // the two warps of these rows
        const float f = row_s[g * 256 + rl];
        named_barrier(pair_bar, 64);
        float m = -INF, l = 0.f;                 // maximum before its factor, sum of this half
        for (int i = 0; i < n; ++i) {
          mbar_wait(&s_full[g], (base + i) & 1, p.err, kErrWait);
          pf_fence_after();
          const int valid = p.prefix_len - (t0 + i) * kPfTokens - half * 64;
          uint32_t pk[32];
          float sum, top;
          // weights against the last maximum; again where the row's largest score of the tile exceeds it by too much
          // (always for the first tile): the scores are in tensor memory until P is written over them
          tile_weights<T>(s_t, valid, m == -INF ? 0.f : m, f, pk, top, sum);
          *mine = top;
          named_barrier(pair_bar, 64);             // both have read their scores, too
          top = fmaxf(top, *other);
          const bool grows = m == -INF ? top != -INF : (top - m) * f > kSlack;
          if (__any_sync(0xffffffffu, grows)) {  // alike in both warps of these rows
            const float nm = fmaxf(m, top);
            if (i) {
              mbar_wait(&pv_done[g], (base + i - 1) & 1, p.err, kErrWait);
              pf_fence_after();
              const float e = m == -INF ? 0.f : fast_exp2((m - nm) * f);
              l *= e;
#pragma unroll 1
              for (int c = 0; c < DV / 64; ++c) {
                float v[32];
                tm_load32(v, o_t + c * 32);
                tm_wait_load(v);
#pragma unroll
                for (int x = 0; x < 32; ++x) v[x] *= e;
                tm_store32(o_t + c * 32, v);
              }
            }
            m = nm;
            tile_weights<T>(s_t, valid, m == -INF ? 0.f : m, f, pk, top, sum);
            named_barrier(pair_bar, 64);           // P of one half lies over scores of the other
          }
          l += sum;
          tm_store32(p_t, pk);
          tm_wait_store();
          pf_fence_before();
          mbar_arrive(&p_ready[g]);
        }
        mbar_wait(&pv_done[g], (base + n - 1) & 1, p.err, kErrWait);
        pf_fence_after();
        *mine = l;
        named_barrier(pair_bar, 64);
        l += *other;
        if (*bad_s) l = __int_as_float(0x7fffffff);
        else if (p.n_heavy && l != l && half == 0 && r0 + r < rows_total) report_dense<D, T>(p, row_of(p, h, 0, r0 + r));
        float* dst = nullptr;
        if (r0 + r < rows_total) {
          if (begins && ends) dst = p.prefix_part + flat_row(p, row_of(p, h, 0, r0 + r)) * RF;
          else dst = p.prefix_slots + ((int64_t)(2 * cta + (begins ? 1 : 0)) * kPfRows + r) * RF;
        }
#pragma unroll 1
        for (int c = 0; c < DV / 64; ++c) {
          float v[32];
          tm_load32(v, o_t + c * 32);
          tm_wait_load(v);
          if (dst) {
#pragma unroll
            for (int x = 0; x < 32; x += 4)
              *reinterpret_cast<float4*>(dst + half * (DV / 2) + c * 32 + x) = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
          }
        }
        if (dst && half == 0) *reinterpret_cast<float2*>(dst + DV) = make_float2(m == -INF ? -INF : m * f - kShift<T>, l);
        pf_fence_before();
      }
      end_piece();
    }
  }
}

constexpr int kPfJoinRows = 8;

// Adds up the pieces of cut items: block (k, .) takes rows of item k, a warp a row.
template <int DV>
__global__ void __launch_bounds__(kPfJoinRows * 32) paged_prefix_join(const __grid_constant__ AttnParams p, int ctas) {
  constexpr int RF = row_floats(DV);
  const int rows_total = p.B * p.G * p.L, items = (rows_total + kPfRows - 1) / kPfRows;
  const int tiles = (p.prefix_len + kPfTokens - 1) / kPfTokens, stride = tiles + kPfItemTiles;
  const int total = stride * items * p.H - kPfItemTiles, grid = min(ctas, total);
  const int h = blockIdx.x / items, r0 = (blockIdx.x - h * items) * kPfRows;
  const int r = blockIdx.y * kPfJoinRows + threadIdx.x / 32, d = (threadIdx.x & 31) * 4;
  asm volatile("griddepcontrol.launch_dependents;");   // the sequences' own tokens need the prefix only where rows are finished
  // by every block: what follows this grid counts on the grid before it, too
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (r0 + r >= rows_total) return;
  // the range that holds a tile of the list: the first total % grid ranges are one longer
  const int q = total / grid, longer = total % grid;
  auto owner = [&](int at) { return at < (q + 1) * longer ? at / (q + 1) : longer + (at - (q + 1) * longer) / q; };
  const int c = owner((int)blockIdx.x * stride), n = owner((int)blockIdx.x * stride + tiles - 1) - c + 1;
  if (n == 1) return;                            // written whole
  float m = -__int_as_float(0x7f800000), l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int k = 0; k < n; ++k) {
    const float* src = p.prefix_slots + ((int64_t)(2 * (c + k) + (k == 0)) * kPfRows + r) * RF;
    const float4 v = d < DV ? *reinterpret_cast<const float4*>(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    join4(m, l, a, src[DV], src[DV + 1], v);
  }
  if (d < DV) finish4<float, DV>(p, row_of(p, h, 0, r0 + r), d, m, l, a);
}

template <int D, int DV, int BD, typename T>
int launch_paged_prefix(const AttnParams& p, const CUtensorMap& vmap, int grid, cudaStream_t st) {
  auto* k = paged_prefix_kernel<D, DV, BD, T>;
  const int smem = PrefixSmem::total(D, DV);
  // the split of registers waits forever where the block has fewer than it was planned for
  static std::atomic<uint64_t> done;
  if (!ready_kernel((const void*)k, smem, kPfLaunchRegs, done))
    return set_last_error(SUNSHAPE_E_CUDA, "the paged prefix kernel is not available as it was built.");
  k<<<grid, kPfThreads, smem, st>>>(p, vmap);
  if (int rc = launch_status("paged prefix launch")) return rc;
  cudaLaunchConfig_t cfg{};
  const int64_t rows = (int64_t)p.B * p.G * p.L;
  cfg.gridDim = dim3((unsigned)((rows + kPfRows - 1) / kPfRows * p.H), kPfRows / kPfJoinRows);
  cfg.blockDim = dim3(kPfJoinRows * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, paged_prefix_join<DV>, p, grid) != cudaSuccess) return launch_status("paged prefix join launch");
  return SUNSHAPE_OK;
}

#define SUNSHAPE_PREFIX_INSTANCE(D, DV, BD, T) \
  template int launch_paged_prefix<D, DV, BD, T>(const AttnParams&, const CUtensorMap&, int, cudaStream_t);
#define SUNSHAPE_PREFIX_INSTANCES(D, T)                                                                             \
  SUNSHAPE_PREFIX_INSTANCE(D, 64, 2, T) SUNSHAPE_PREFIX_INSTANCE(D, 64, 4, T) SUNSHAPE_PREFIX_INSTANCE(D, 64, 8, T) \
  SUNSHAPE_PREFIX_INSTANCE(D, 128, 2, T) SUNSHAPE_PREFIX_INSTANCE(D, 128, 4, T) SUNSHAPE_PREFIX_INSTANCE(D, 128, 8, T)

}  // namespace sunshape
