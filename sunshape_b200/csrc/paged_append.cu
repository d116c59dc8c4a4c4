// Append to a paged compressed cache: rotate, permute and encode keys, copy values, into token slots.
//
// index = argmin_c |z_b - C_b[c]|^2 for block b of the rotated, permuted key z.  The choice is made exactly:
// a scan in fp32 of  |c|^2 - 2 z.c  (|z|^2 is common to all codewords) keeps the smallest and the second
// smallest value, whose errors against real arithmetic are below E (see kBound); where they lie within 2 E of
// each other the block is decided by a scan in 64 bits.
#include "paged.cuh"

namespace sunshape {
namespace {

struct AppendParams {
  const void* key;
  const void* val;
  int64_t ks[3], vs[3];       // strides of (b, h, l), elements
  int L, H, D, Dv, nb, bd, C, n_cb, ps, n_heavy;
  int64_t tokens, slots_total;
  const int64_t* slots;
  int64_t slot_sb, slot_sl;
  const float* cb;
  const int64_t* perm;
  const uint8_t* heavy_mask;
  uint8_t* idx;
  void* heavy;
  void* out_val;
  Rotation rot;
  int* err;
};

// The fp32 scan's error: z rounded to fp32 (relative u = 2^-24), bd products summed by fma, |c|^2 summed by
// fma, one last fma: at most u (bd + 2) (|c|^2 + 2 |z| |c|) <= 10 u (...) for bd <= 8; 16 covers the terms of
// second order and the rounding of the bound itself, kTiny what underflows.
constexpr float kBound = 16.f / 16777216.f;
constexpr float kTiny = 1e-37f;

constexpr int kTokens = 64;   // tokens of a CTA
constexpr int kLanes = 4;     // threads that share a token's codewords

// element d of the rotated key in 64 bits: the products of a 16-bit by a 24-bit significand are exact
template <typename T>
__device__ __forceinline__ double rotated(const AppendParams& p, const T* row, int d, int64_t pos) {
  const double y = (double)Elem<T>::to_float(row[d]);
  if (d >= p.rot.rot) return y;
  int other, i;
  bool second;
  pair_of(p.rot, d, other, i, second);
  const double o = (double)Elem<T>::to_float(row[other]);
  const double c = (double)p.rot.cos[pos * (p.rot.rot / 2) + i], s = (double)p.rot.sin[pos * (p.rot.rot / 2) + i];
  return second ? y * c + o * s : y * c - o * s;
}

// slot of a token, -1 where it is left out; records what is out of range
__device__ __forceinline__ int64_t slot_of(const AppendParams& p, int64_t b, int64_t l, int64_t& pos) {
  int64_t slot = p.slots[b * p.slot_sb + l * p.slot_sl];
  if (slot < -1 || slot >= p.slots_total) {
    record_error(p.err, kErrSlot);
    slot = -1;
  }
  pos = 0;
  if (slot >= 0 && p.rot.rot) {
    pos = position_of(p.rot, b, l);
    if (pos < 0 || pos >= p.rot.table_len) {
      record_error(p.err, kErrPosition);
      slot = -1;
    }
  }
  return slot;
}

// grid (token tiles, heads, blocks + 1): the last z copies the values
template <typename T, int BD>
__global__ void __launch_bounds__(kTokens * kLanes) append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ __align__(16) float cb_s[256 * BD];
  __shared__ float cn_s[256];
  __shared__ int cmax_s;
  const int tid = threadIdx.x, h = blockIdx.y, blk = blockIdx.z;
  const int64_t t = (int64_t)blockIdx.x * kTokens + tid / kLanes;
  const int s = tid % kLanes;
  int64_t b = 0, l = 0, slot = -1, pos = 0;
  if (t < p.tokens) {
    b = t / p.L;
    l = t - b * p.L;
    slot = slot_of(p, b, l, pos);
  }
  const int64_t row = slot < 0 ? 0 : (slot / p.ps * p.H + h) * p.ps + slot % p.ps;   // page row of this head
  if (blk == p.nb) {
    if (slot < 0) return;
    const T* src = reinterpret_cast<const T*>(p.val) + b * p.vs[0] + h * p.vs[1] + l * p.vs[2];
    T* dst = reinterpret_cast<T*>(p.out_val) + row * p.Dv;
    if ((uintptr_t)src % 16 == 0) {
      for (int i = s; i < p.Dv / 8; i += kLanes)
        reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(src)[i];
    } else {
      for (int i = s; i < p.Dv; i += kLanes) dst[i] = src[i];
    }
    return;
  }
  const T* krow = reinterpret_cast<const T*>(p.key) + b * p.ks[0] + h * p.ks[1] + l * p.ks[2];
  if (p.heavy_mask && p.heavy_mask[blk]) {
    if (slot < 0) return;
    int at = 0;
    for (int i = 0; i < blk; ++i) at += p.heavy_mask[i] != 0;
    T* dst = reinterpret_cast<T*>(p.heavy) + (row * p.n_heavy + at) * BD;
    for (int w = s; w < BD; w += kLanes)
      dst[w] = Elem<T>::from_float((float)rotated(p, krow, (int)p.perm[blk * BD + w], pos));
    if (s == 0) p.idx[row * p.nb + blk] = 0;
    return;
  }
  const float* cb = p.cb + ((int64_t)(p.n_cb == 1 ? 0 : h % p.n_cb) * p.nb + blk) * p.C * BD;
  if (tid == 0) cmax_s = 0;
  for (int i = tid; i < p.C * BD; i += blockDim.x) cb_s[i] = cb[i];
  __syncthreads();
  for (int c = tid; c < p.C; c += blockDim.x) {
    float n = 0.f;
#pragma unroll
    for (int w = 0; w < BD; ++w) n = fmaf(cb_s[c * BD + w], cb_s[c * BD + w], n);
    cn_s[c] = n;
    atomicMax(&cmax_s, __float_as_int(n));       // not negative: ordered as integers; NaN above all
  }
  __syncthreads();
  const float INF = __int_as_float(0x7f800000);
  double z[BD];
  float x[BD], zn = 0.f;
#pragma unroll
  for (int w = 0; w < BD; ++w) {
    z[w] = slot < 0 ? 0.0 : rotated(p, krow, (int)p.perm[blk * BD + w], pos);
    x[w] = (float)z[w];
    zn = fmaf(x[w], x[w], zn);
  }
  float best = INF, next = INF;
  int at = p.C;
  for (int c = s; c < p.C; c += kLanes) {
    float dot = 0.f;
#pragma unroll
    for (int w = 0; w < BD; ++w) dot = fmaf(x[w], cb_s[c * BD + w], dot);
    const float d = fmaf(-2.f, dot, cn_s[c]);
    if (d < best) {
      next = best;
      best = d;
      at = c;
    } else {
      next = fminf(next, d);
    }
  }
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) {
    const float ob = __shfl_xor_sync(0xffffffffu, best, o), on = __shfl_xor_sync(0xffffffffu, next, o);
    const int oa = __shfl_xor_sync(0xffffffffu, at, o);
    next = fminf(fminf(next, on), fmaxf(best, ob));
    if (ob < best) {
      best = ob;
      at = oa;
    }
  }
  const float cm2 = __int_as_float(cmax_s);
  const float E = kBound * (cm2 + 2.f * sqrtf(zn) * sqrtf(cm2)) + kTiny;
  const bool unsure = slot >= 0 && !(next - best > 2.f * E);    // NaN and infinities are unsure
  if (__any_sync(0xffffffffu, unsure)) {
    double bd64 = __longlong_as_double(0x7ff0000000000000ll);
    int a64 = p.C;
    if (unsure) {
      for (int c = s; c < p.C; c += kLanes) {
        double d = 0.0;
#pragma unroll
        for (int w = 0; w < BD; ++w) {
          const double e = z[w] - (double)cb_s[c * BD + w];
          d = fma(e, e, d);
        }
        if (d < bd64) {
          bd64 = d;
          a64 = c;
        }
      }
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) {
      const double od = __shfl_xor_sync(0xffffffffu, bd64, o);
      const int oa = __shfl_xor_sync(0xffffffffu, a64, o);
      if (od < bd64 || (od == bd64 && oa < a64)) {
        bd64 = od;
        a64 = oa;
      }
    }
    if (unsure) at = a64;
  }
  if (slot >= 0 && s == 0) p.idx[row * p.nb + blk] = (uint8_t)(at < p.C ? at : 0);   // no finite distance: 0
}

template <typename T>
void launch(const AppendParams& p, cudaStream_t st) {
  const dim3 grid((unsigned)((p.tokens + kTokens - 1) / kTokens), p.H, p.nb + 1);
  if (p.bd == 8) append_kernel<T, 8><<<grid, kTokens * kLanes, 0, st>>>(p);
  else if (p.bd == 4) append_kernel<T, 4><<<grid, kTokens * kLanes, 0, st>>>(p);
  else append_kernel<T, 2><<<grid, kTokens * kLanes, 0, st>>>(p);
}

}  // namespace

int check_pages(const sunshape_codec_t* c, const sunshape_pages_t* pg) {
  if (int rc = check_codec_args(c)) return rc;
  if (!pg) return set_last_error(SUNSHAPE_E_INVALID, "page pool descriptor is NULL.");
  if (c->block_dim != 2 && c->block_dim != 4 && c->block_dim != 8)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "the paged cache takes block_dim 2, 4 or 8.");
  if (c->n_centroids > 256)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "the paged cache takes at most 256 codewords a block.");
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

extern "C" int sunshape_paged_append(const sunshape_codec_t* codec, const sunshape_pages_t* pages,
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
  if (!key->data || !value->data || !slots) return set_last_error(SUNSHAPE_E_INVALID, "key / value / slots pointer is NULL.");
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
  p.bd = codec->block_dim;
  p.nb = p.D / p.bd;
  p.C = codec->n_centroids;
  p.n_cb = codec->n_cb;
  p.ps = pages->page_size;
  p.n_heavy = codec->heavy_mask ? codec->n_heavy : 0;
  p.slots_total = pages->num_pages * pages->page_size;
  p.slots = slots;
  p.slot_sb = slot_stride_b;
  p.slot_sl = slot_stride_l;
  p.cb = codec->centroids;
  p.perm = codec->permutation;
  p.heavy_mask = p.n_heavy ? codec->heavy_mask : nullptr;
  p.idx = pages->indices;
  p.heavy = pages->heavy;
  p.out_val = pages->value;
  p.err = paged_error_word();
  if (!p.err) return set_last_error(SUNSHAPE_E_CUDA, "the paged error word is unavailable on this device.");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (pages->dtype == SUNSHAPE_BF16) launch<__nv_bfloat16>(p, st);
  else launch<__half>(p, st);
  return launch_status("paged append launch");
}
