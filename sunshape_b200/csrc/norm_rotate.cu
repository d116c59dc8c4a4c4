// Head norms of queries and keys with the position rotation in the same pass.
//
//   y = x * w / sqrt(mean(x^2) + eps),   z_i = y_i c_i - y_j s_i,   z_j = y_j c_i + y_i s_i
//
// Bound by memory: every row is read and written once, and the pass does about ten fp32 operations an
// element.  A row is 256 bytes at dim 128, so one thread takes 16 elements of a row as two 16-byte loads that
// hold whole pairs (elements 8s .. 8s+7 of each half, or 16s .. 16s+15 when neighbours pair up): the rotation
// then needs no exchange between threads, only the norm's sum does (three shuffles at dim 128).  Cosines and
// sines belong to the token, not to the head, so a thread keeps them in registers over the heads that it takes.
// Measured on B200: 69 us for 16384 tokens of 40 heads of 128 in bf16 (344 MB, 5.0 TB/s, 76 % of a copy); with four heads a
// group of threads and no rows in flight beyond them 88 us; 3.0 us for 8 tokens of 72 heads.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "paged.cuh"

namespace sunshape {
namespace {

struct NormRotateParams {
  const void* x[2];
  void* y[2];
  int64_t xs[2][3], ys[2][3];   // strides of (b, h, l), elements
  int heads[2];
  const void* w[2];
  int w_dtype, w_vec;           // w_vec: weights are 16-byte aligned
  float eps;
  int L, dim, width;            // width: threads of a row (vector kernel)
  int parts;                    // groups of threads that share a token's heads
  int64_t tokens, items;
  Rotation rot;
  int* err;
};

template <typename T>
struct Vec8 {
  uint4 v[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, Vec8<T>& r) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
}

template <typename T>
__device__ __forceinline__ void unpack8(const Vec8<T>& r, float* f) {
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = Elem<T>::to_float(e[i]);
}

// two fp32 numbers as a pair of 16-bit ones, in one instruction
template <typename T>
__device__ __forceinline__ uint32_t pair_of_floats(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* f) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pair_of_floats<T>(f[0], f[1]), pair_of_floats<T>(f[2], f[3]),
                                              pair_of_floats<T>(f[4], f[5]), pair_of_floats<T>(f[6], f[7]));
  }
}

// eight weights from element e on (a multiple of eight)
__device__ __forceinline__ void load_weights(const void* w, int e, int dtype, bool vec, float* f) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = load_as_float(w, e + i, dtype);
  } else if (dtype == SUNSHAPE_F32) {
    Vec8<float> r;
    load8(reinterpret_cast<const float*>(w) + e, r);
    unpack8(r, f);
  } else if (dtype == SUNSHAPE_BF16) {
    Vec8<__nv_bfloat16> r;
    load8(reinterpret_cast<const __nv_bfloat16*>(w) + e, r);
    unpack8(r, f);
  } else {
    Vec8<__half> r;
    load8(reinterpret_cast<const __half*>(w) + e, r);
    unpack8(r, f);
  }
}

// A group of `width` threads takes every `parts`th head of a token -- so that neighbouring groups touch neighbouring
// rows -- with the next four rows always in flight.
template <typename T, bool INTER>
__global__ void __launch_bounds__(128) norm_rotate_vec(const __grid_constant__ NormRotateParams p) {
  constexpr int N = 4;
  const int W = p.width;
  const int s = threadIdx.x & (W - 1);
  const unsigned item = (blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32) * (32 / W) + (threadIdx.x & 31) / W;
  if (item >= (unsigned)p.items) return;  // whole groups leave: the shuffles below stay within a group
  const unsigned mask = W == 32 ? 0xffffffffu : ((1u << W) - 1) << ((threadIdx.x & 31) & ~(W - 1));
  const unsigned token = item / (unsigned)p.parts;
  const int64_t b = token / (unsigned)p.L, l = token - (unsigned)b * (unsigned)p.L;
  const bool have = s * 16 < p.dim;       // the last threads of a group are idle when dim / 16 is no power of two
  const int R = p.rot.rot;
  const bool turned = s * 16 < R;
  // first elements of this thread's two runs of eight
  const int e0 = !INTER && turned ? 8 * s : 16 * s;
  const int e1 = !INTER && turned ? 8 * s + R / 2 : 16 * s + 8;
  int h = (int)(item - token * (unsigned)p.parts);

  for (int which = 0; which < 2; ++which) {
    const int heads = p.heads[which];
    if (h >= heads) {
      h -= heads;
      continue;
    }
    const T* x = reinterpret_cast<const T*>(p.x[which]) + b * p.xs[which][0] + l * p.xs[which][2];
    T* y = reinterpret_cast<T*>(p.y[which]) + b * p.ys[which][0] + l * p.ys[which][2];
    const int64_t x_step = p.xs[which][1], y_step = p.ys[which][1];
    Vec8<T> in[N][2];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (have && h + i * p.parts < heads) {
        load8(x + (h + i * p.parts) * x_step + e0, in[i][0]);
        load8(x + (h + i * p.parts) * x_step + e1, in[i][1]);
      }
    }
    // Of the pairs' elements (u, v) come u A - v B and v C + u S: the rotation with the weights multiplied in, once for
    // all of the thread's heads.  A thread's pairs are (e0 + e, e1 + e), or neighbours in its sixteen elements.
    float A[8], B[8], C[8], S[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) A[e] = C[e] = 1.f, B[e] = S[e] = 0.f;
    const void* w = p.w[which];
    if (w && have) {
      float w0[8], w1[8];
      load_weights(w, e0, p.w_dtype, p.w_vec, w0);
      load_weights(w, e1, p.w_dtype, p.w_vec, w1);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        A[e] = INTER ? (e < 4 ? w0[2 * e & 7] : w1[2 * e & 7]) : w0[e];
        C[e] = INTER ? (e < 4 ? w0[(2 * e + 1) & 7] : w1[(2 * e + 1) & 7]) : w1[e];
      }
    }
    bool bad = false;
    if (R) {
      const int64_t pos = position_of(p.rot, b, l);
      bad = pos < 0 || pos >= p.rot.table_len;
      if (bad && s == 0) record_error(p.err, kErrPosition);
      if (turned) {
        const int64_t at = (bad ? 0 : pos) * (R / 2) + 8 * s;
        float c[8], sn[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          reinterpret_cast<float4*>(c)[i] = reinterpret_cast<const float4*>(p.rot.cos + at)[i];
          reinterpret_cast<float4*>(sn)[i] = reinterpret_cast<const float4*>(p.rot.sin + at)[i];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          S[e] = A[e] * sn[e];
          B[e] = C[e] * sn[e];
          A[e] *= c[e];
          C[e] *= c[e];
        }
      }
    }
    while (h < heads) {
#pragma unroll
      for (int i = 0; i < N; ++i, h += p.parts) {
        if (h >= heads) break;                // the same for the whole group
        float a0[8], a1[8];
        unpack8(in[i][0], a0);
        unpack8(in[i][1], a1);
        if (have && h + N * p.parts < heads) {
          load8(x + (h + N * p.parts) * x_step + e0, in[i][0]);
          load8(x + (h + N * p.parts) * x_step + e1, in[i][1]);
        }
        float r = 1.f;
        if (w) {
          float q = 0.f;
          if (have) {
#pragma unroll
            for (int e = 0; e < 8; ++e) q = fmaf(a0[e], a0[e], fmaf(a1[e], a1[e], q));
          }
          for (int o = W >> 1; o; o >>= 1) q += __shfl_xor_sync(mask, q, o);
          r = rsqrtf(q / (float)p.dim + p.eps);
        }
        if (bad) r = __int_as_float(0x7fffffff);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float& u = INTER ? (e < 4 ? a0[2 * e & 7] : a1[2 * e & 7]) : a0[e];
          float& v = INTER ? (e < 4 ? a0[(2 * e + 1) & 7] : a1[(2 * e + 1) & 7]) : a1[e];
          float zu = u * A[e], zv = v * C[e];
          if (turned) {                       // not as products with zero: elements beyond R keep to themselves
            zu = fmaf(-v, B[e], zu);
            zv = fmaf(u, S[e], zv);
          }
          u = zu * r;
          v = zv * r;
        }
        if (have) {
          store8(y + h * y_step + e0, a0);
          store8(y + h * y_step + e1, a1);
        }
      }
    }
    h -= heads;
  }
}

// Any dim, rot_dim, stride and alignment: one warp a row, the row staged in shared memory so that it may be
// overwritten in place.
template <typename T>
__global__ void __launch_bounds__(128) norm_rotate_any(const __grid_constant__ NormRotateParams p) {
  extern __shared__ float rows[];
  const int lane = threadIdx.x & 31;
  float* f = rows + (threadIdx.x >> 5) * p.dim;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= p.items) return;
  const int per = p.heads[0] + p.heads[1];
  const int64_t token = row / per;
  int h = (int)(row - token * per);
  const int which = h >= p.heads[0];
  if (which) h -= p.heads[0];
  const int64_t b = token / p.L, l = token - b * p.L;
  const T* x = reinterpret_cast<const T*>(p.x[which]) + b * p.xs[which][0] + h * p.xs[which][1] + l * p.xs[which][2];
  T* y = reinterpret_cast<T*>(p.y[which]) + b * p.ys[which][0] + h * p.ys[which][1] + l * p.ys[which][2];
  float q = 0.f;
  for (int d = lane; d < p.dim; d += 32) {
    const float v = Elem<T>::to_float(x[d]);
    f[d] = v;
    q = fmaf(v, v, q);
  }
  __syncwarp();
  if (p.w[which]) {
    for (int o = 16; o; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
    const float r = rsqrtf(q / (float)p.dim + p.eps);
    for (int d = lane; d < p.dim; d += 32) f[d] = f[d] * r * load_as_float(p.w[which], d, p.w_dtype);
    __syncwarp();
  }
  int64_t pos = 0;
  bool bad = false;
  if (p.rot.rot) {
    pos = position_of(p.rot, b, l);
    bad = pos < 0 || pos >= p.rot.table_len;
    if (bad && lane == 0) record_error(p.err, kErrPosition);
    if (bad) pos = 0;
  }
  for (int d = lane; d < p.dim; d += 32) {
    float v = f[d];
    if (d < p.rot.rot) {
      int other, i;
      bool second;
      pair_of(p.rot, d, other, i, second);
      const float c = p.rot.cos[pos * (p.rot.rot / 2) + i], sn = p.rot.sin[pos * (p.rot.rot / 2) + i];
      v = second ? v * c + f[other] * sn : v * c - f[other] * sn;
    }
    y[d] = Elem<T>::from_float(bad ? __int_as_float(0x7fffffff) : v);
  }
}

template <typename T>
void launch(NormRotateParams& p, bool vec, cudaStream_t st) {
  if (!vec) {
    p.items = p.tokens * (p.heads[0] + p.heads[1]);
    norm_rotate_any<T><<<(unsigned)((p.items + 3) / 4), 128, 4 * p.dim * sizeof(float), st>>>(p);
    return;
  }
  int w = 1;
  while (w * 16 < p.dim) w *= 2;
  p.width = w;
  // Groups that share a token: one where there are tokens enough to give every SM 512 threads, which a thread's cosines,
  // weights and rows in flight allow; up to one for each head below that, so that a decode step's few rows spread out.
  const int heads = p.heads[0] + p.heads[1];
  p.parts = (int)std::min<int64_t>(heads, std::max<int64_t>(1, (int64_t)paged_sm_count() * 512 / w / p.tokens));
  p.items = p.tokens * p.parts;
  const unsigned grid = (unsigned)((p.items * w + 127) / 128);
  if (p.rot.interleaved) norm_rotate_vec<T, true><<<grid, 128, 0, st>>>(p);
  else norm_rotate_vec<T, false><<<grid, 128, 0, st>>>(p);
}

bool float_type(int d) { return d == SUNSHAPE_F32 || d == SUNSHAPE_BF16 || d == SUNSHAPE_F16; }

}  // namespace

__device__ int g_paged_error;

int* paged_error_word() {
  static std::atomic<int*> known[64];            // the address of a device's word never changes
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return nullptr;
  int* w = dev < 64 ? known[dev].load(std::memory_order_relaxed) : nullptr;
  if (w) return w;
  void* a = nullptr;
  if (cudaGetSymbolAddress(&a, g_paged_error) != cudaSuccess) return nullptr;
  if (dev < 64) known[dev].store(static_cast<int*>(a), std::memory_order_relaxed);
  return static_cast<int*>(a);
}

int paged_sm_count() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return sm_count();
  int n = known[dev].load(std::memory_order_relaxed);
  if (!n) known[dev].store(n = sm_count(), std::memory_order_relaxed);
  return n;
}

bool ready_kernel(const void* kernel, int smem, int regs, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (dev < 64 && done.load(std::memory_order_acquire) >> dev & 1) return true;
  if (regs) {
    cudaFuncAttributes a;
    if (cudaFuncGetAttributes(&a, kernel) != cudaSuccess || a.numRegs != regs) return false;
  }
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return false;
  if (dev < 64) done.fetch_or(uint64_t(1) << dev, std::memory_order_release);
  return true;
}

int make_rotation(const sunshape_rotation_t* r, int dim, bool empty, Rotation* out) {
  *out = Rotation{};
  if (!r || r->rot_dim == 0) return SUNSHAPE_OK;
  if (r->rot_dim < 0 || r->rot_dim > dim || r->rot_dim % 2)
    return set_last_error(SUNSHAPE_E_INVALID, "rot_dim must be even and between 0 and the head dimension.");
  if (!empty && (!r->cos || !r->sin || !r->positions)) return set_last_error(SUNSHAPE_E_INVALID, "rotation pointer is NULL.");
  if (r->table_len < 0) return set_last_error(SUNSHAPE_E_INVALID, "rotation table length must be >= 0.");
  // the kernels read row 0 where a position is outside the table
  if (!empty && r->table_len == 0) return set_last_error(SUNSHAPE_E_INVALID, "the rotation table has no rows.");
  if (r->position_dtype != SUNSHAPE_I32 && r->position_dtype != SUNSHAPE_I64)
    return set_last_error(SUNSHAPE_E_INVALID, "positions must be I32 or I64.");
  *out = Rotation{r->cos, r->sin, r->positions, r->position_stride_b, r->position_stride_l, r->table_len,
                  r->position_dtype == SUNSHAPE_I64, r->rot_dim, r->interleaved != 0};
  return SUNSHAPE_OK;
}

}  // namespace sunshape

using namespace sunshape;

extern "C" {

int sunshape_paged_error(int32_t* code, int32_t clear) {
  if (!code) return set_last_error(SUNSHAPE_E_INVALID, "code pointer is NULL.");
  int* w = paged_error_word();
  // the copy alone would not wait for streams that do not block the default one
  if (!w || cudaDeviceSynchronize() != cudaSuccess || cudaMemcpy(code, w, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess)
    return set_last_error(SUNSHAPE_E_CUDA, "reading the paged error word failed.");
  // A word that holds a code takes no other one, so a clear loses none; one that holds none is not cleared, and a
  // clear is done before the call returns.
  if (clear && *code && (cudaMemset(w, 0, sizeof(int)) != cudaSuccess || cudaStreamSynchronize(nullptr) != cudaSuccess))
    return set_last_error(SUNSHAPE_E_CUDA, "clearing the paged error word failed.");
  return SUNSHAPE_OK;
}

int sunshape_norm_rotate(const sunshape_rows_t* q, const sunshape_rows_t* q_out, const void* q_weight,
                         const sunshape_rows_t* k, const sunshape_rows_t* k_out, const void* k_weight, int32_t dtype,
                         int32_t weight_dtype, int32_t batch, int32_t length, int32_t dim, float eps,
                         const sunshape_rotation_t* rotation, void* stream) {
  if (!q || !q_out) return set_last_error(SUNSHAPE_E_INVALID, "query rows descriptor is NULL.");
  if (!k != !k_out) return set_last_error(SUNSHAPE_E_INVALID, "key rows need both an input and an output.");
  if (!float_type(dtype)) return set_last_error(SUNSHAPE_E_INVALID, "row dtype must be F32, BF16 or F16.");
  if ((q_weight || k_weight) && !float_type(weight_dtype))
    return set_last_error(SUNSHAPE_E_INVALID, "norm weight dtype must be F32, BF16 or F16.");
  if (batch < 0 || length < 0 || dim < 1 || dim > 2048)
    return set_last_error(SUNSHAPE_E_INVALID, "batch and length must be >= 0 and the head dimension 1 to 2048.");
  NormRotateParams p{};
  if (int rc = make_rotation(rotation, dim, batch == 0 || length == 0, &p.rot)) return rc;
  const sunshape_rows_t* in[2] = {q, k};
  const sunshape_rows_t* out[2] = {q_out, k_out};
  const int size = dtype == SUNSHAPE_F32 ? 4 : 2, unit = 16 / size;
  bool vec = dim % 16 == 0 && dim <= 512 && p.rot.rot % 16 == 0 && ((uintptr_t)p.rot.cos | (uintptr_t)p.rot.sin) % 16 == 0;
  p.w[0] = q_weight;
  p.w[1] = k_weight;
  for (int i = 0; i < 2 && in[i]; ++i) {
    if (in[i]->heads < 0 || in[i]->heads != out[i]->heads)
      return set_last_error(SUNSHAPE_E_INVALID, "input and output rows must have the same number of heads.");
    if (in[i]->heads && (!in[i]->data || !out[i]->data) && batch && length)
      return set_last_error(SUNSHAPE_E_INVALID, "rows pointer is NULL.");
    p.x[i] = in[i]->data;
    p.y[i] = out[i]->data;
    p.heads[i] = in[i]->heads;
    const int64_t a[3] = {in[i]->stride_b, in[i]->stride_h, in[i]->stride_l};
    const int64_t b[3] = {out[i]->stride_b, out[i]->stride_h, out[i]->stride_l};
    for (int j = 0; j < 3; ++j) {
      p.xs[i][j] = a[j];
      p.ys[i][j] = b[j];
      vec = vec && a[j] % unit == 0 && b[j] % unit == 0;
    }
    vec = vec && ((uintptr_t)p.x[i] | (uintptr_t)p.y[i]) % 16 == 0;
  }
  p.tokens = (int64_t)batch * length;
  if (p.tokens * (p.heads[0] + p.heads[1]) == 0) return SUNSHAPE_OK;
  if (p.tokens * (p.heads[0] + p.heads[1]) > (int64_t)1 << 31)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "at most 2^31 rows a call.");
  p.w_dtype = weight_dtype;
  p.w_vec = ((uintptr_t)q_weight | (uintptr_t)k_weight) % 16 == 0;
  p.eps = eps;
  p.L = length;
  p.dim = dim;
  p.err = paged_error_word();
  if (!p.err) return set_last_error(SUNSHAPE_E_CUDA, "the paged error word is unavailable on this device.");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == SUNSHAPE_F32) launch<float>(p, vec, st);
  else if (dtype == SUNSHAPE_BF16) launch<__nv_bfloat16>(p, vec, st);
  else launch<__half>(p, vec, st);
  return launch_status("norm_rotate launch");
}

}  // extern "C"
