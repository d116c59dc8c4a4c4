// Append to a paged compressed cache: rotate, permute and encode keys, copy values, into token slots.
//
// index = argmin_c |z_b - C_b[c]|^2 = argmax_c z_b.C_b[c] - |C_b[c]|^2 / 2  for block b of the rotated, permuted
// key z, decided exactly in three steps of growing precision:
//   1. on the tensor cores, z and c as sums of two fp16 numbers and -|c|^2 / 2 as the accumulator's start, every
//      thread keeps the maximum of each group of 16 codewords that it sees.  Where one group alone comes within
//      twice the error bound of the overall maximum, the answer is in it;
//   2. its 16 codewords (otherwise all) are compared in fp32, keeping the smallest and the second smallest distance.
//      Where they differ by more than twice the error bound, the smallest is the answer;
//   3. otherwise (borders between codewords, repeated codewords, infinities and NaN) a warp scans the block in 64 bits.
//
// Bound by instructions: 256 distances for every block against 2 (D + Dv) bytes a key and head.  Step 1 takes per 16
// tokens x 8 codewords one or two MMAs and four maxima -- comparing all in fp32 takes 8 multiply-adds and 3 comparisons a
// distance.  Measured on B200: 4096 tokens of 8 heads, 32 blocks of 4: 90 us (all in fp32: 242); 5425 tokens of 8 heads,
// 12 blocks of 8 and 4 dense ones: 109 us (246); 64 tokens of 8 heads, 16 blocks of 8: 8.7 us (17.4).
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace sunshape {
namespace {

struct AppendParams {
  const void* key;
  const void* val;
  int64_t ks[3], vs[3];       // strides of (b, h, l), elements
  int L, H, D, Dv, nb, C, n_cb, ps, n_heavy;
  int blocks, splits;         // blocks of a CTA, CTAs that share a head's blocks
  int64_t tokens, slots_total;
  const int64_t* slots;
  int64_t slot_sb, slot_sl;
  const uint8_t* records;
  const int64_t* perm;
  const uint8_t* heavy_mask;
  uint8_t* idx;
  void* heavy;
  void* out_val;
  Rotation rot;
  int* err;
};

// Step 1's error is below filter(BD) (|z| + 0.5), the block's scale bringing |c| below 1: of the products' and the
// start's sum, every addend may be cut to 2^-23 of the largest (|z| or 0.5; BD 8: 25 addends in two steps, BD 4: 13, BD
// 2: 7, and one rounding a step), and z and c are off by at most 2^-22 of themselves, or 2^-25, and the product of their
// remainders is left out: four times 2^-22 |z| for all of these.
// That addends are cut no further is what B200 does, not what is documented: over 168 million scores a block_dim (keys and
// codewords of equal and of unequal sizes, one sign, every low bit set, cancelling ones) the largest error was 0.07, 0.11 and
// 0.15 of the bound at BD 8, 4 and 2.
__host__ __device__ constexpr float filter(int bd) { return (bd == 8 ? 28 + 8 : bd == 4 ? 14 + 8 : 8 + 8) * 1.1f / 8388608.f; }
// Step 2's: d = sum (c - z)^2 in fp32 is off by at most (bd + 3) u d (u = 2^-24) for its own roundings, and by
// 2 sqrt(d) r + r^2 for z being off by r <= 2 u |z| + 4 u^2 |y| (see rotate32; |y|: the key's largest element).  kBound
// covers bd <= 8, terms of second order and the rounding of the bound itself, kTiny what underflows.
constexpr float kUlp = 1.f / 16777216.f, kBound = 16.f * kUlp, kTiny = 1e-37f;

constexpr int kWarps = 4;
constexpr int kTokens = 32 * kWarps;   // tokens of a CTA: two groups of 16 a warp

// element d of the rotated key in 64 bits: the products of a 16-bit by a 24-bit significand are exact
template <typename T>
__device__ __forceinline__ double rotated(const Rotation& r, const T* row, int d, int64_t pos) {
  const double y = (double)Elem<T>::to_float(row[d]);
  if (d >= r.rot) return y;
  int other, i;
  bool second;
  pair_of(r, d, other, i, second);
  const double o = (double)Elem<T>::to_float(row[other]);
  const double c = (double)r.cos[pos * (r.rot / 2) + i], s = (double)r.sin[pos * (r.rot / 2) + i];
  return second ? y * c + o * s : y * c - o * s;
}

// the same in fp32, y c -+ o s with the rounding of the second product taken back: off by at most two roundings of
// the result and of 2^-24 of that product
__device__ __forceinline__ float rotate32(float y, float o, float c, float s) {
  const float q = o * s, e = fmaf(o, s, -q);
  return fmaf(y, c, q) + e;
}

// slot of a token, -1 where it is left out; records what is out of range
__device__ __forceinline__ int64_t slot_of(const AppendParams& p, int64_t b, int64_t l, int64_t& pos) {
  int64_t slot = p.slots[b * p.slot_sb + l * p.slot_sl];
  pos = p.rot.rot ? position_of(p.rot, b, l) : 0;
  if (slot < -1 || slot >= p.slots_total) {
    record_error(p.err, kErrSlot);
    slot = -1;
  }
  if (slot >= 0 && p.rot.rot && (pos < 0 || pos >= p.rot.table_len)) {
    record_error(p.err, kErrPosition);
    slot = -1;
  }
  return slot;
}

// d = a b + (start of each column, the same in all rows) -- or + c
__device__ __forceinline__ void mma_k16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, float2 c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y));
}
__device__ __forceinline__ void mma_k8(float* d, uint32_t a0, uint32_t a1, uint32_t b0, float2 c) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%8,%7,%8};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0), "f"(c.x), "f"(c.y));
}
__device__ __forceinline__ void mma_k8(float* d, uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0));
}

// Whether a result of rotate32, off by two units of its last place, may round to T otherwise than the exact one, itself
// rounded to fp32 first (as torch rounds 64 bits to 16): it
// lies near the middle of two neighbours, is below f16's normal range, or so much smaller than the key's largest element
// that the second product's error counts.
template <typename T>
__device__ __forceinline__ bool near_tie(float z, float most) {
  constexpr int LOW = std::is_same<T, __half>::value ? 13 : 16;
  const int off = (__float_as_int(z) & ((1 << LOW) - 1)) - (1 << (LOW - 1));
  return abs(off) <= 8 || !(fabsf(z) > most * (1.f / 1048576.f)) || (LOW == 13 && fabsf(z) < 6.2e-5f);
}

// for error bounds, which have room for its own error of 2^-22
__device__ __forceinline__ float sqrt_approx(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// a block's elements, aligned to 16 bytes (8 for two)
template <int BD>
__device__ __forceinline__ void load_block(const float* p, float* v) {
  if constexpr (BD == 2) {
    *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < BD / 4; ++i) reinterpret_cast<float4*>(v)[i] = reinterpret_cast<const float4*>(p)[i];
  }
}

// two fp32 numbers as a pair of fp16 and the pair of their remainders
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const __half2 l = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Which codewords of a lane's fragment row: the contraction of a block is over its BD elements, z_hi c_hi + z_lo c_hi +
// z_hi c_lo, laid into the MMA's K:
//   BD 8: one k16 step [z_hi | z_lo] [c_hi | c_hi] and one k8 step z_hi c_lo
//   BD 4: one k16 step [z_hi | z_lo | z_hi | 0] [c_hi | c_hi | c_lo | 0]
//   BD 2: one k8 step  [z_hi | z_lo | z_hi | 0] [c_hi | c_hi | c_lo | 0]

// Codebooks into the attention image and the encoder's fragments: a CTA a block, a thread a codeword.
template <int BD>
__global__ void __launch_bounds__(256) tables_kernel(const float* cb, const float* norm_max, bool dense, int C, int nb,
                                                     int D, uint8_t* out, Tables at) {
  __shared__ float red[256];
  __shared__ float v_s[256][BD];
  const int blk = blockIdx.x, k = blockIdx.y, c = threadIdx.x;
  const float* block = cb + ((int64_t)k * nb + blk) * C * BD;
  float n = 0.f;
#pragma unroll
  for (int w = 0; w < BD; ++w) {
    v_s[c][w] = c < C ? block[c * BD + w] : 0.f;
    n = fmaf(v_s[c][w], v_s[c][w], n);
  }
  // largest norm of the block, and of the codebook where the caller did not give it
  float all = n;
  if (!norm_max)
    for (int i = c; i < nb * C; i += 256) {
      float m = 0.f;
      for (int w = 0; w < BD; ++w) {
        const float v = cb[((int64_t)k * nb * C + i) * BD + w];
        m = fmaf(v, v, m);
      }
      all = fmaxf(all, m);
    }
  auto most = [&](float v) {
    __syncthreads();
    red[c] = v;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
      if (c < o) red[c] = fmaxf(red[c], red[c + o]);
      __syncthreads();
    }
    return red[0];
  };
  // the power of two that brings a norm into [0.5, 1); 1 for 0
  auto factor = [](float norm) {
    if (!(norm > 0.f)) return 1.f;
    int e;
    frexpf(norm, &e);
    return ldexpf(1.f, -max(-100, min(100, e)));
  };
  const float bs = factor(sqrtf(most(n)));
  // at most 1 beside dense blocks, which are read in the same scale: all of fp16 stays in reach
  const float is = fminf(factor(norm_max ? norm_max[k] : sqrtf(most(all))), dense ? 1.f : 2e30f);
  constexpr int PER = 64 / BD;      // blocks of an image row
  __half* image = reinterpret_cast<__half*>(out) +
                  (((int64_t)k * ((D + 63) / 64) + blk / PER) * 256 + c) * 64 + blk % PER * BD;
#pragma unroll
  for (int w = 0; w < BD; ++w) image[w] = __float2half_rn(v_s[c][w] * is);
  uint8_t* rec = out + at.records + ((int64_t)k * nb + blk) * record_bytes(BD);
  reinterpret_cast<float*>(rec + kRecNorms)[c] = c < C ? -0.5f * (n * bs) * bs : -1e30f;
#pragma unroll
  for (int w = 0; w < BD; ++w) reinterpret_cast<float*>(rec + kRecWords)[c * BD + w] = c < C ? v_s[c][w] : 1e18f;
  if (c < 4) reinterpret_cast<float*>(rec + kRecWords + 1024 * BD)[c] = c == 0 ? bs : 0.f;
  if (c == 0 && blk == 0) reinterpret_cast<float*>(out + at.iscale)[k] = is;
  uint2* frags = reinterpret_cast<uint2*>(rec);
  for (int i = c; i < 1024; i += 256) {
    const int word = i >> 5, g = (i & 31) >> 2, t = i & 3;
    const float* v = v_s[word * 8 + g];
    uint32_t hi, lo;
    uint2 f = make_uint2(0u, 0u);
    if constexpr (BD == 8) {
      split2(v[2 * t] * bs, v[2 * t + 1] * bs, hi, lo);
      f = make_uint2(hi, lo);
    } else if constexpr (BD == 4) {
      split2(v[2 * (t & 1)] * bs, v[2 * (t & 1) + 1] * bs, hi, lo);
      f = make_uint2(hi, t < 2 ? lo : 0u);
    } else {
      split2(v[0] * bs, v[1] * bs, hi, lo);
      f = make_uint2(t < 2 ? hi : (t == 2 ? lo : 0u), 0u);
    }
    frags[i] = f;
  }
}

// grid (token tiles, heads, splits + 1): the last z copies the values
template <typename T, int BD>
__global__ void __launch_bounds__(kWarps * 32) append_kernel(const __grid_constant__ AppendParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int REC = record_bytes(BD);
  const int width = p.blocks * BD, ld = width + 8;                 // permuted elements of this CTA, row stride
  uint8_t* const rec_s = smem;                                     // [2][REC]
  float* const z_s = reinterpret_cast<float*>(rec_s + 2 * REC);    // [kTokens][ld]
  int64_t* const slot_s = reinterpret_cast<int64_t*>(z_s + kTokens * ld);   // [kTokens] page row of this head, -1: left out
  int64_t* const pos_s = slot_s + kTokens;
  int64_t* const key_s = pos_s + kTokens;                          // offset of the key row
  int* const most_s = reinterpret_cast<int*>(key_s + kTokens);     // [kTokens] largest element of the key, as an integer
  uint8_t* const idx_s = reinterpret_cast<uint8_t*>(most_s + kTokens);   // [kTokens][blocks]
  __shared__ uint64_t bar_s[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y;
  const int64_t t0 = (int64_t)blockIdx.x * kTokens;
  const int n_tok = (int)min((int64_t)kTokens, p.tokens - t0);
  const bool values = blockIdx.z == p.splits;
  if (tid < kTokens) {
    int64_t slot = -1, pos = 0, at = 0;
    if (tid < n_tok) {
      const int64_t b = (t0 + tid) / p.L, l = t0 + tid - b * p.L;
      slot = slot_of(p, b, l, pos);
      if (slot >= 0) slot = (slot / p.ps * p.H + h) * p.ps + slot % p.ps;
      at = values ? b * p.vs[0] + h * p.vs[1] + l * p.vs[2] : b * p.ks[0] + h * p.ks[1] + l * p.ks[2];
    }
    slot_s[tid] = slot;
    pos_s[tid] = slot < 0 ? 0 : pos;            // rows that are left out are read, not used
    key_s[tid] = at;
    most_s[tid] = 0;
  }
  __syncthreads();
  if (values) {
    const T* const v = reinterpret_cast<const T*>(p.val);
    T* const out = reinterpret_cast<T*>(p.out_val);
    const int per = p.Dv / 8;
    for (int i = tid; i < n_tok * per; i += kWarps * 32) {
      const int tok = i / per, d = (i - tok * per) * 8;
      if (slot_s[tok] < 0) continue;
      const T* src = v + key_s[tok] + d;
      T* dst = out + slot_s[tok] * p.Dv + d;
      if ((uintptr_t)src % 16 == 0) {
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
      } else {
        for (int j = 0; j < 8; ++j) dst[j] = src[j];
      }
    }
    return;
  }
  const int b0 = blockIdx.z * p.blocks, nblk = min(p.blocks, p.nb - b0);
  const uint8_t* const records = p.records + ((int64_t)(p.n_cb == 1 ? 0 : h % p.n_cb) * p.nb + b0) * REC;
  if (tid == 0) {                               // the first two blocks' records
    for (int i = 0; i < 2; ++i) mbar_init(&bar_s[i], 1);
    fence_mbar_init();
    for (int i = 0; i < min(2, nblk); ++i) {
      mbar_arrive_expect_tx(&bar_s[i], REC);
      bulk_g2s(rec_s + i * REC, records + (int64_t)i * REC, REC, &bar_s[i]);
    }
  }
  const T* const keys = reinterpret_cast<const T*>(p.key);
  {
    // rotated keys: a thread keeps its column of the permuted rows and takes every `step`th token
    const int step = kWarps * 32 / width;       // blocks are chosen so that width is at most the threads
    const int e = tid % width;
    if (tid < step * width && e < nblk * BD) {
      const int d = (int)p.perm[b0 * BD + e];
      int other = d, i = 0;
      bool second = false;
      const bool turned = d < p.rot.rot;
      if (turned) pair_of(p.rot, d, other, i, second);
      const int half = p.rot.rot / 2;
      constexpr int N = 8;                      // tokens in flight
      for (int first = tid / width; first < n_tok; first += N * step) {
        float y[N], o[N], c[N], sn[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int tok = min(first + k * step, n_tok - 1);
          const T* row = keys + key_s[tok];
          y[k] = Elem<T>::to_float(row[d]);
          o[k] = 0.f;
          if (turned) {
            o[k] = Elem<T>::to_float(row[other]);
            c[k] = p.rot.cos[pos_s[tok] * half + i];
            sn[k] = p.rot.sin[pos_s[tok] * half + i];
          }
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int tok = first + k * step;
          if (tok >= n_tok) break;
          // not negative: ordered as integers, NaN above all
          const int size = max(__float_as_int(fabsf(y[k])), __float_as_int(fabsf(o[k])));
          if (size > most_s[tok]) atomicMax(&most_s[tok], size);
          z_s[tok * ld + e] = turned ? rotate32(y[k], o[k], c[k], second ? sn[k] : -sn[k]) : y[k];
        }
      }
    }
  }
  const int g = lane >> 2, t = lane & 3;
  const float INF = __int_as_float(0x7f800000);
  const int w0 = warp * 32;                     // the warp's first token
  __syncthreads();

  for (int j = 0; j < nblk; ++j) {
    const int blk = b0 + j;
    uint8_t* const rec = rec_s + (j & 1) * REC;
    mbar_wait(&bar_s[j & 1], (j >> 1) & 1, p.err, kErrWait);
    if (p.heavy_mask && p.heavy_mask[blk]) {
      int at = 0;
      for (int i = 0; i < blk; ++i) at += p.heavy_mask[i] != 0;
      for (int i = tid; i < n_tok * BD; i += kWarps * 32) {
        const int tok = i / BD, w = i % BD;
        if (slot_s[tok] < 0) continue;
        float z = z_s[tok * ld + j * BD + w];
        if (near_tie<T>(z, __int_as_float(most_s[tok])))
          z = (float)rotated(p.rot, keys + key_s[tok], (int)p.perm[blk * BD + w], pos_s[tok]);
        reinterpret_cast<T*>(p.heavy)[(slot_s[tok] * p.n_heavy + at) * BD + w] = Elem<T>::from_float(z);
      }
      if (tid < n_tok) idx_s[tid * p.blocks + j] = 0;
    } else if (w0 < n_tok) {
      const uint2* const frag_s = reinterpret_cast<const uint2*>(rec);
      const float* const norm_s = reinterpret_cast<const float*>(rec + kRecNorms);
      const float* const cb_s = reinterpret_cast<const float*>(rec + kRecWords);
      const float scale = cb_s[256 * BD];
      // ---- step 1
      uint32_t a[2][4], a8[2][2];
      float bound[2][2];                                             // twice the error of rows g and g + 8
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float* z = z_s + min(w0 + mt * 16 + y * 8 + g, n_tok - 1) * ld + j * BD;
          alignas(16) float x[BD];
          load_block<BD>(z, x);
          float q = 0.f;
#pragma unroll
          for (int w = 0; w < BD; ++w) q = fmaf(x[w] * scale, x[w] * scale, q);
          bound[mt][y] = 2.f * filter(BD) * (sqrt_approx(q) + 0.5f);
          uint32_t hi, lo;
          const int e = BD == 8 ? 2 * t : (BD == 4 ? 2 * (t & 1) : 0);
          split2(z[e] * scale, z[e + 1] * scale, hi, lo);
          if constexpr (BD == 8) {
            a[mt][y] = hi;
            a[mt][2 + y] = lo;
            a8[mt][y] = hi;
          } else if constexpr (BD == 4) {
            a[mt][y] = t < 2 ? hi : lo;
            a[mt][2 + y] = t < 2 ? hi : 0u;
          } else {
            a8[mt][y] = t == 1 ? lo : (t == 3 ? 0u : hi);
          }
        }
      }
      float top[2][2][4];                                            // maxima of groups of eight n-tiles
#pragma unroll
      for (int grp = 0; grp < 4; ++grp) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) top[mt][0][grp] = top[mt][1][grp] = -INF;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int nt = grp * 8 + i;
          const uint2 f = frag_s[nt * 32 + lane];
          const float2 nn = *reinterpret_cast<const float2*>(norm_s + nt * 8 + 2 * t);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            float s[4];
            if constexpr (BD == 8) {
              mma_k16(s, a[mt], f.x, f.x, nn);
              mma_k8(s, a8[mt][0], a8[mt][1], f.y);
            } else if constexpr (BD == 4) {
              mma_k16(s, a[mt], f.x, f.y, nn);
            } else {
              mma_k8(s, a8[mt][0], a8[mt][1], f.x, nn);
            }
            top[mt][0][grp] = fmaxf(top[mt][0][grp], fmaxf(s[0], s[1]));
            top[mt][1][grp] = fmaxf(top[mt][1][grp], fmaxf(s[2], s[3]));
          }
        }
      }
      // the group of 16 codewords (lane of the quad, n-tile group) that alone is near the maximum; -1: there are several
      int where[2][2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float m = fmaxf(fmaxf(top[mt][y][0], top[mt][y][1]), fmaxf(top[mt][y][2], top[mt][y][3]));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          int v = 0;                                               // number of groups, and the sum of what names them
#pragma unroll
          for (int grp = 0; grp < 4; ++grp)
            if (top[mt][y][grp] >= m - bound[mt][y]) v += 256 + (grp * 4 + t);
          v += __shfl_xor_sync(0xffffffffu, v, 1);
          v += __shfl_xor_sync(0xffffffffu, v, 2);
          // -2: a bound that is no number, or a key beyond fp16 in the block's scale
          where[mt][y] = !(bound[mt][y] < 2.f * filter(BD) * 30000.f) ? -2 : ((v >> 8) == 1 ? v & 255 : -1);
        }
      // ---- step 2: a lane a token
      const int tok = w0 + lane, from = (lane & 7) * 4;
      int found = __shfl_sync(0xffffffffu, where[0][0], from);
      const int f01 = __shfl_sync(0xffffffffu, where[0][1], from), f10 = __shfl_sync(0xffffffffu, where[1][0], from);
      const int f11 = __shfl_sync(0xffffffffu, where[1][1], from);
      if (lane & 16) found = lane & 8 ? f11 : f10;
      else if (lane & 8) found = f01;
      const bool live = tok < n_tok && slot_s[min(tok, n_tok - 1)] >= 0;
      alignas(16) float x[BD];
      float zn = 0.f, best = INF, next = INF;
      int at = p.C;
      load_block<BD>(z_s + min(tok, n_tok - 1) * ld + j * BD, x);
#pragma unroll
      for (int w = 0; w < BD; ++w) zn = fmaf(x[w], x[w], zn);
      if (found >= 0) {
        const int c0 = (found >> 2) * 64 + 2 * (found & 3);
        const float* v = cb_s + c0 * BD;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int c = (i >> 1) * 8 + (i & 1);
          alignas(16) float u[BD];
          float d = 0.f;
          load_block<BD>(v + c * BD, u);
#pragma unroll
          for (int w = 0; w < BD; ++w) d = fmaf(u[w] - x[w], u[w] - x[w], d);
          next = fminf(next, fmaxf(best, d));
          if (d < best) {
            best = d;
            at = c0 + c;
          }
        }
      }
      // several groups near the maximum: the warp compares all of the block's codewords
      unsigned wide = __ballot_sync(0xffffffffu, live && found == -1);
      for (; wide; wide &= wide - 1) {
        const int who = __ffs(wide) - 1;
        alignas(16) float xw[BD];
        float near1 = INF, near2 = INF;
        int c1 = p.C;
        load_block<BD>(z_s + (w0 + who) * ld + j * BD, xw);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          alignas(16) float u[BD];
          float d = 0.f;
          load_block<BD>(cb_s + (i * 32 + lane) * BD, u);
#pragma unroll
          for (int w = 0; w < BD; ++w) d = fmaf(u[w] - xw[w], u[w] - xw[w], d);
          near2 = fminf(near2, fmaxf(near1, d));
          if (d < near1) {
            near1 = d;
            c1 = i * 32 + lane;
          }
        }
        const float mine = near1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float n1 = __shfl_xor_sync(0xffffffffu, near1, o), n2 = __shfl_xor_sync(0xffffffffu, near2, o);
          near2 = fminf(fminf(near2, n2), fmaxf(near1, n1));
          near1 = fminf(near1, n1);
        }
        const unsigned at1 = __ballot_sync(0xffffffffu, mine == near1);   // one lane, unless step 3 decides
        c1 = __shfl_sync(0xffffffffu, c1, at1 ? __ffs(at1) - 1 : 0);
        if (lane == who) {
          best = near1;
          next = near2;
          at = c1;
        }
      }
      const float rz = 4.f * kUlp * sqrt_approx(zn) + 16.f * kUlp * kUlp * __int_as_float(most_s[min(tok, n_tok - 1)]);
      const float E = kBound * next + 4.f * rz * (sqrt_approx(next) + rz) + kTiny;
      // ---- step 3; also where a codeword that is none was the nearest (keys that lie where those are kept)
      unsigned unsure = __ballot_sync(0xffffffffu, live && !(found > -2 && at < p.C && next - best > 2.f * E));
      for (; unsure; unsure &= unsure - 1) {
        const int who = __ffs(unsure) - 1, tk = w0 + who;
        double zz[BD], bd64 = __longlong_as_double(0x7ff0000000000000ll);
        int a64 = p.C;
#pragma unroll
        for (int w = 0; w < BD; ++w)
          zz[w] = rotated(p.rot, keys + key_s[tk], (int)p.perm[blk * BD + w], pos_s[tk]);
        for (int c = lane; c < p.C; c += 32) {
          double d = 0.0;
#pragma unroll
          for (int w = 0; w < BD; ++w) {
            const double e = zz[w] - (double)cb_s[c * BD + w];
            d = fma(e, e, d);
          }
          if (d < bd64) {
            bd64 = d;
            a64 = c;
          }
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double od = __shfl_xor_sync(0xffffffffu, bd64, o);
          const int oc = __shfl_xor_sync(0xffffffffu, a64, o);
          if (od < bd64 || (od == bd64 && oc < a64)) {
            bd64 = od;
            a64 = oc;
          }
        }
        if (lane == who) at = a64;
      }
      if (live) idx_s[tok * p.blocks + j] = (uint8_t)(at < p.C ? at : 0);   // no finite distance: 0
    }
    __syncthreads();                            // the record is read
    if (tid == 0 && j + 2 < nblk) {
      mbar_arrive_expect_tx(&bar_s[j & 1], REC);
      bulk_g2s(rec, records + (int64_t)(j + 2) * REC, REC, &bar_s[j & 1]);
    }
  }
  if (p.blocks % 4 == 0 && p.nb % 4 == 0) {
    const int per = nblk / 4;
    for (int i = tid; i < n_tok * per; i += kWarps * 32) {
      const int tok = i / per, q = i - tok * per;
      if (slot_s[tok] >= 0)
        reinterpret_cast<uint32_t*>(p.idx + slot_s[tok] * p.nb + b0)[q] =
            reinterpret_cast<const uint32_t*>(idx_s + tok * p.blocks)[q];
    }
  } else {
    for (int i = tid; i < n_tok * nblk; i += kWarps * 32) {
      const int tok = i / nblk, q = i - tok * nblk;
      if (slot_s[tok] >= 0) p.idx[slot_s[tok] * p.nb + b0 + q] = idx_s[tok * p.blocks + q];
    }
  }
}

template <typename T, int BD>
int launch(AppendParams& p, cudaStream_t st) {
  const int64_t tiles = (p.tokens + kTokens - 1) / kTokens;
  // A head's blocks are shared out until every SM has two CTAs (one token a sequence leaves one tile of tokens), and in
  // any case to 32 elements a CTA, with whose keys in shared memory an SM holds five
  const int64_t fill = 2 * paged_sm_count() / (tiles * p.H);
  p.blocks = (int)std::min<int64_t>((p.nb + std::max<int64_t>(fill, 1) - 1) / std::max<int64_t>(fill, 1), 32 / BD);
  p.splits = (p.nb + p.blocks - 1) / p.blocks;
  const int smem = 2 * record_bytes(BD) + kTokens * ((p.blocks * BD + 8) * 4 + 3 * 8 + 4 + p.blocks);
  static std::atomic<uint64_t> done;
  if (!ready_kernel((const void*)append_kernel<T, BD>, 2 * record_bytes(BD) + kTokens * (40 * 4 + 28 + 32 / BD), 0, done))
    return set_last_error(SUNSHAPE_E_CUDA, "the paged append kernel is not available as it was built.");
  append_kernel<T, BD><<<dim3((unsigned)tiles, p.H, p.splits + 1), kWarps * 32, smem, st>>>(p);
  return launch_status("paged append launch");
}

template <typename T>
int launch(AppendParams& p, int bd, cudaStream_t st) {
  if (bd == 8) return launch<T, 8>(p, st);
  return bd == 4 ? launch<T, 4>(p, st) : launch<T, 2>(p, st);
}

int check_paged_codec(const sunshape_codec_t* c) {
  if (int rc = check_codec_args(c)) return rc;
  if (c->block_dim != 2 && c->block_dim != 4 && c->block_dim != 8)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "the paged cache takes block_dim 2, 4 or 8.");
  if (c->n_centroids > 256)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "the paged cache takes at most 256 codewords a block.");
  return SUNSHAPE_OK;
}

}  // namespace

int check_pages(const sunshape_codec_t* c, const sunshape_pages_t* pg) {
  if (int rc = check_paged_codec(c)) return rc;
  if (!pg) return set_last_error(SUNSHAPE_E_INVALID, "page pool descriptor is NULL.");
  if (pg->dtype != SUNSHAPE_BF16 && pg->dtype != SUNSHAPE_F16)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "the paged cache holds BF16 or F16 values.");
  if (pg->kv_heads < 1 || pg->kv_heads > 65535 || pg->num_pages < 0 || pg->page_size < 16 || pg->page_size % 16 ||
      pg->value_dim < 8 || pg->value_dim % 8)
    return set_last_error(SUNSHAPE_E_INVALID, "page pool: kv_heads 1 to 65535, page_size a multiple of 16 and "
                                              "value_dim a multiple of 8 are required.");
  if (pg->num_pages > 0 && (!pg->indices || !pg->value))
    return set_last_error(SUNSHAPE_E_INVALID, "page pool pointer is NULL.");
  if (c->heavy_mask && c->n_heavy > 0 && pg->num_pages > 0 && !pg->heavy)
    return set_last_error(SUNSHAPE_E_INVALID, "page pool: a codec with dense blocks needs a heavy pool.");
  if (((uintptr_t)pg->indices | (uintptr_t)pg->value | (uintptr_t)pg->heavy) % 16)
    return set_last_error(SUNSHAPE_E_INVALID, "page pools must be 16-byte aligned.");
  return SUNSHAPE_OK;
}

}  // namespace sunshape

using namespace sunshape;

extern "C" {

int64_t sunshape_paged_tables_bytes(const sunshape_codec_t* codec) {
  if (int rc = check_paged_codec(codec)) return rc;
  return Tables(codec->n_cb, codec->head_dim / codec->block_dim, codec->head_dim).total;
}

int sunshape_paged_tables(const sunshape_codec_t* codec, void* tables, int64_t tables_bytes, void* stream) {
  if (int rc = check_paged_codec(codec)) return rc;
  const int nb = codec->head_dim / codec->block_dim;
  const Tables at(codec->n_cb, nb, codec->head_dim);
  if (!tables || (uintptr_t)tables % 256 || tables_bytes < at.total)
    return set_last_error(SUNSHAPE_E_INVALID, "tables buffer missing, misaligned or too small.");
  if (codec->n_cb > 65535) return set_last_error(SUNSHAPE_E_UNSUPPORTED, "at most 65535 codebooks.");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(nb, codec->n_cb);
  uint8_t* out = static_cast<uint8_t*>(tables);
#define SUNSHAPE_TABLES_CASE(BD)                                                                                     \
  if (codec->block_dim == BD)                                                                                        \
    tables_kernel<BD><<<grid, 256, 0, st>>>(codec->centroids, codec->centroid_norm_max,                              \
                                            codec->heavy_mask && codec->n_heavy > 0, codec->n_centroids, nb,         \
                                            codec->head_dim, out, at);
  SUNSHAPE_TABLES_CASE(2)
  SUNSHAPE_TABLES_CASE(4)
  SUNSHAPE_TABLES_CASE(8)
#undef SUNSHAPE_TABLES_CASE
  return launch_status("paged tables launch");
}

int sunshape_paged_append(const sunshape_codec_t* codec, const void* tables, const sunshape_pages_t* pages,
                                     const sunshape_rows_t* key, const sunshape_rows_t* value, int32_t batch,
                                     int32_t length, const int64_t* slots, int64_t slot_stride_b,
                                     int64_t slot_stride_l, const sunshape_rotation_t* rotation, void* stream) {
  if (int rc = check_pages(codec, pages)) return rc;
  if (!key || !value) return set_last_error(SUNSHAPE_E_INVALID, "key / value rows descriptor is NULL.");
  if (batch < 0 || length < 0) return set_last_error(SUNSHAPE_E_INVALID, "batch and length must be >= 0.");
  if (key->heads != pages->kv_heads || value->heads != pages->kv_heads)
    return set_last_error(SUNSHAPE_E_INVALID, "key and value rows must have the pool's kv_heads.");
  AppendParams p{};
  if (int rc = make_rotation(rotation, codec->head_dim, batch == 0 || length == 0, &p.rot)) return rc;
  p.tokens = (int64_t)batch * length;
  if (p.tokens == 0) return SUNSHAPE_OK;
  if (!key->data || !value->data || !slots || !tables)
    return set_last_error(SUNSHAPE_E_INVALID, "key / value / slots pointer or tables are NULL.");
  if (p.tokens > (int64_t)1 << 30) return set_last_error(SUNSHAPE_E_UNSUPPORTED, "at most 2^30 rows a call.");
  p.key = key->data;
  p.val = value->data;
  const int64_t ks[3] = {key->stride_b, key->stride_h, key->stride_l};
  const int64_t vs[3] = {value->stride_b, value->stride_h, value->stride_l};
  for (int i = 0; i < 3; ++i) {
    p.ks[i] = ks[i];
    p.vs[i] = vs[i];
  }
  p.L = length;
  p.H = pages->kv_heads;
  p.D = codec->head_dim;
  p.Dv = pages->value_dim;
  p.nb = p.D / codec->block_dim;
  p.C = codec->n_centroids;
  p.n_cb = codec->n_cb;
  p.ps = pages->page_size;
  p.n_heavy = codec->heavy_mask ? codec->n_heavy : 0;
  p.slots_total = pages->num_pages * pages->page_size;
  p.slots = slots;
  p.slot_sb = slot_stride_b;
  p.slot_sl = slot_stride_l;
  const Tables tab(p.n_cb, p.nb, p.D);
  p.records = static_cast<const uint8_t*>(tables) + tab.records;
  p.perm = codec->permutation;
  p.heavy_mask = p.n_heavy ? codec->heavy_mask : nullptr;
  p.idx = pages->indices;
  p.heavy = pages->heavy;
  p.out_val = pages->value;
  p.err = paged_error_word();
  if (!p.err) return set_last_error(SUNSHAPE_E_CUDA, "the paged error word is unavailable on this device.");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return pages->dtype == SUNSHAPE_BF16 ? launch<__nv_bfloat16>(p, codec->block_dim, st) : launch<__half>(p, codec->block_dim, st);
}

}  // extern "C"
