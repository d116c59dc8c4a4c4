// Attention of decode steps over a paged compressed cache, with an optional prefix that the batch shares.
//
//   o = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),   s_t = scale <q, k_hat_t>,   m = max_t s_t
//
// The tokens of a sequence are cut into runs; a CTA computes (m, l, acc) of 16 query rows over one run and a
// second kernel joins the runs of a row.
#include "paged.cuh"

namespace sunshape {
namespace {

constexpr int kRows = 16;       // query rows of a CTA
constexpr int kTile = 32;       // tokens of a step
constexpr int kRun = 512;       // tokens of a run
constexpr int kThreads = 128;

struct AttnParams {
  const void* q;
  int64_t qs[3];
  int B, Hq, H, L, G, D, Dv, nb, bd, C, n_cb, ps, n_heavy, cols, prefix, causal, runs, mtiles;
  int64_t num_pages, table_stride;
  float scale;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* prefix_table;
  const float* cb;
  const int64_t* perm;
  const uint8_t* heavy_mask;
  const uint8_t* idx;
  const void* heavy;
  const void* val;
  void* out;
  float* part;                  // [runs][B * Hq * L][2 + Dv]
  int* err;
};

// length of sequence b's own tokens; -1 where the call is invalid
__device__ __forceinline__ int own_length(const AttnParams& p, int b) {
  const int n = p.lens[b];
  return n < 0 || n > (int64_t)p.cols * p.ps ? -1 : n;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) attention_simple(const __grid_constant__ AttnParams p) {
  extern __shared__ float sm[];
  float* q_s = sm;                                  // [16][D]
  float* k_s = q_s + kRows * p.D;                   // [32][D + 1]
  float* v_s = k_s + kTile * (p.D + 1);             // [32][Dv]
  float* p_s = v_s + kTile * p.Dv;                  // [16][33]
  float* m_s = p_s + kRows * (kTile + 1);           // [16] max, sum, factor
  float* l_s = m_s + kRows;
  float* f_s = l_s + kRows;
  __shared__ int64_t row_s[kTile];
  __shared__ int bad_s;
  const float INF = __int_as_float(0x7f800000);
  const int tid = threadIdx.x, run = blockIdx.x, h = blockIdx.y / p.mtiles, mt = blockIdx.y % p.mtiles, b = blockIdx.z;
  const int rows = p.G * p.L, r0 = mt * kRows, nr = min(kRows, rows - r0);
  const int own = own_length(p, b);
  if (own < 0 && run == 0 && tid == 0) record_error(p.err, kErrLength);
  const int total = own < 0 ? 0 : p.prefix + own;
  const int t0 = run * kRun, t1 = min(total, t0 + kRun);
  if (tid == 0) bad_s = own < 0;
  for (int i = tid; i < nr * p.D; i += kThreads) {
    const int r = r0 + i / p.D, d = i % p.D;
    const int hq = h * p.G + r / p.L, l = r % p.L;
    q_s[i] = Elem<T>::to_float(reinterpret_cast<const T*>(p.q)[b * p.qs[0] + hq * p.qs[1] + l * p.qs[2] + p.perm[d]]);
  }
  if (tid < kRows) {
    m_s[tid] = -INF;
    l_s[tid] = 0.f;
  }
  const int per = kThreads / p.Dv == 0 ? 1 : kThreads / p.Dv;   // threads of one output column (Dv 64 or 128)
  const int col = tid % p.Dv, rg = tid / p.Dv;
  float acc[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) acc[i] = 0.f;
  __syncthreads();
  for (int t = t0; t < t1; t += kTile) {
    const int nt = min(kTile, t1 - t);
    if (tid < nt) {
      const int tok = t + tid;
      const int at = tok < p.prefix ? tok : tok - p.prefix;
      const int page = tok < p.prefix ? p.prefix_table[at / p.ps] : p.table[b * p.table_stride + at / p.ps];
      if (page < 0 || page >= p.num_pages) {
        record_error(p.err, kErrPage);
        bad_s = 1;
        row_s[tid] = -1;
      } else {
        row_s[tid] = ((int64_t)page * p.H + h) * p.ps + at % p.ps;
      }
    }
    __syncthreads();
    for (int i = tid; i < nt * p.nb; i += kThreads) {
      const int n = i / p.nb, bl = i % p.nb;
      const int64_t row = row_s[n];
      if (row < 0) continue;
      float* dst = k_s + n * (p.D + 1) + bl * p.bd;
      if (p.heavy_mask && p.heavy_mask[bl]) {
        int at = 0;
        for (int j = 0; j < bl; ++j) at += p.heavy_mask[j] != 0;
        for (int w = 0; w < p.bd; ++w)
          dst[w] = Elem<T>::to_float(reinterpret_cast<const T*>(p.heavy)[(row * p.n_heavy + at) * p.bd + w]);
      } else {
        const int c = min((int)p.idx[row * p.nb + bl], p.C - 1);
        const float* src = p.cb + (((int64_t)(p.n_cb == 1 ? 0 : h % p.n_cb) * p.nb + bl) * p.C + c) * p.bd;
        for (int w = 0; w < p.bd; ++w) dst[w] = src[w];
      }
    }
    for (int i = tid; i < nt * p.Dv; i += kThreads) {
      const int64_t row = row_s[i / p.Dv];
      v_s[i] = row < 0 ? 0.f : Elem<T>::to_float(reinterpret_cast<const T*>(p.val)[row * p.Dv + i % p.Dv]);
    }
    __syncthreads();
    for (int i = tid; i < kRows * kTile; i += kThreads) {
      const int r = i / kTile, n = i % kTile;
      float s = -INF;
      // query l sees all but the last L - 1 - l of the sequence's own tokens
      const int seen = p.prefix + (p.causal ? max(0, own - (p.L - 1 - (r0 + r) % p.L)) : own);
      if (r < nr && n < nt && t + n < seen) {
        s = 0.f;
        for (int d = 0; d < p.D; ++d) s = fmaf(q_s[r * p.D + d], k_s[n * (p.D + 1) + d], s);
        s *= p.scale * kLog2e;
      }
      p_s[r * (kTile + 1) + n] = s;
    }
    __syncthreads();
    if (tid < kRows) {
      float m = m_s[tid];
      for (int n = 0; n < kTile; ++n) m = fmaxf(m, p_s[tid * (kTile + 1) + n]);
      const float base = m == -INF ? 0.f : m;
      float l = 0.f;
      for (int n = 0; n < kTile; ++n) {
        const float e = exp2f(p_s[tid * (kTile + 1) + n] - base);
        p_s[tid * (kTile + 1) + n] = e;
        l += e;
      }
      f_s[tid] = exp2f(m_s[tid] - base);
      l_s[tid] = l_s[tid] * f_s[tid] + l;
      m_s[tid] = m;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (i % per != rg) continue;
      float a = acc[i] * f_s[i];
      for (int n = 0; n < nt; ++n) a = fmaf(p_s[i * (kTile + 1) + n], v_s[n * p.Dv + col], a);
      acc[i] = a;
    }
    __syncthreads();
  }
  const bool bad = bad_s != 0;
  for (int i = 0; i < kRows; ++i) {
    if (i >= nr || i % per != rg) continue;
    const int r = r0 + i, hq = h * p.G + r / p.L, l = r % p.L;
    float* dst = p.part + ((int64_t)run * p.B * p.Hq * p.L + ((int64_t)b * p.Hq + hq) * p.L + l) * (2 + p.Dv);
    dst[2 + col] = bad ? __int_as_float(0x7fffffff) : acc[i];
    if (col == 0) {
      dst[0] = bad ? 0.f : m_s[i];
      dst[1] = bad ? 1.f : l_s[i];
    }
  }
}

template <typename T>
__global__ void join_simple(const __grid_constant__ AttnParams p) {
  const float INF = __int_as_float(0x7f800000);
  const int64_t row = blockIdx.x, rows = (int64_t)p.B * p.Hq * p.L;
  const int own = own_length(p, (int)(row / ((int64_t)p.Hq * p.L)));
  const int used = own < 0 ? 1 : max(1, (p.prefix + own + kRun - 1) / kRun);
  float m = -INF;
  for (int k = 0; k < used; ++k) m = fmaxf(m, p.part[(k * rows + row) * (2 + p.Dv)]);
  const float base = m == -INF ? 0.f : m;
  float l = 0.f, a = 0.f;
  for (int k = 0; k < used; ++k) {
    const float* src = p.part + (k * rows + row) * (2 + p.Dv);
    const float f = exp2f(src[0] - base);
    l = fmaf(src[1], f, l);
    a = fmaf(src[2 + threadIdx.x], f, a);
  }
  reinterpret_cast<T*>(p.out)[row * p.Dv + threadIdx.x] = Elem<T>::from_float(l > 0.f ? a / l : (l == 0.f ? 0.f : l));
}

template <typename T>
void launch(const AttnParams& p, cudaStream_t st) {
  const int smem = (kRows * p.D + kTile * (p.D + 1) + kTile * p.Dv + kRows * (kTile + 1) + 3 * kRows) * 4;
  cudaFuncSetAttribute(attention_simple<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  attention_simple<T><<<dim3(p.runs, p.H * p.mtiles, p.B), kThreads, smem, st>>>(p);
  join_simple<T><<<(unsigned)((int64_t)p.B * p.Hq * p.L), p.Dv, 0, st>>>(p);
}

int64_t max_runs(int64_t cols, int64_t ps, int64_t prefix) {
  const int64_t n = (cols * ps + prefix + kRun - 1) / kRun;
  return n < 1 ? 1 : n;
}

}  // namespace
}  // namespace sunshape

using namespace sunshape;

extern "C" {

int64_t sunshape_paged_attention_workspace_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t query_len,
                                                 int32_t value_dim, int32_t table_cols, int32_t page_size,
                                                 int32_t prefix_len) {
  (void)kv_heads;
  return max_runs(table_cols, page_size, prefix_len) * batch * q_heads * query_len * (2 + value_dim) * 4;
}

int sunshape_paged_attention(const sunshape_codec_t* codec, const sunshape_pages_t* pages, const void* codebook,
                             const float* codebook_scale, const sunshape_rows_t* query, int32_t batch,
                             int32_t query_len, const int32_t* page_table, int64_t table_stride, int32_t table_cols,
                             const int32_t* seq_lens, const int32_t* prefix_table, int32_t prefix_len, float scale,
                             int32_t causal, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_pages(codec, pages)) return rc;
  if (!query) return set_last_error(SUNSHAPE_E_INVALID, "query rows descriptor is NULL.");
  if (codec->head_dim != 64 && codec->head_dim != 128)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "paged attention takes head_dim 64 or 128.");
  if (pages->value_dim != 64 && pages->value_dim != 128)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "paged attention takes value_dim 64 or 128.");
  if (batch < 0 || query_len < 0 || query->heads < 0 || table_cols < 0 || prefix_len < 0)
    return set_last_error(SUNSHAPE_E_INVALID, "negative size.");
  if (query->heads % pages->kv_heads)
    return set_last_error(SUNSHAPE_E_INVALID, "Query head count must be divisible by kv-head count.");
  if ((int64_t)table_cols * pages->page_size > (int64_t)1 << 30 || prefix_len > 1 << 30)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "at most 2^30 tokens a sequence.");
  const int64_t rows = (int64_t)batch * query->heads * query_len;
  if (rows == 0) return SUNSHAPE_OK;
  if (batch > 65535 || rows > (int64_t)1 << 30)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "at most 65535 sequences and 2^30 query rows a call.");
  if (!query->data || !out || !seq_lens || (table_cols && !page_table) || (prefix_len && !prefix_table) || !codebook ||
      !codebook_scale)
    return set_last_error(SUNSHAPE_E_INVALID, "query / out / seq_lens / page table / codebook pointer is NULL.");
  if (!workspace || (uintptr_t)workspace % 256 ||
      workspace_bytes < sunshape_paged_attention_workspace_bytes(batch, query->heads, pages->kv_heads, query_len,
                                                                 pages->value_dim, table_cols, pages->page_size,
                                                                 prefix_len))
    return set_last_error(SUNSHAPE_E_WORKSPACE, "paged attention: workspace missing, misaligned or too small.");
  AttnParams p{};
  p.q = query->data;
  p.qs[0] = query->stride_b;
  p.qs[1] = query->stride_h;
  p.qs[2] = query->stride_l;
  p.B = batch;
  p.Hq = query->heads;
  p.H = pages->kv_heads;
  p.L = query_len;
  p.G = p.Hq / p.H;
  p.D = codec->head_dim;
  p.Dv = pages->value_dim;
  p.bd = codec->block_dim;
  p.nb = p.D / p.bd;
  p.C = codec->n_centroids;
  p.n_cb = codec->n_cb;
  p.ps = pages->page_size;
  p.n_heavy = codec->heavy_mask ? codec->n_heavy : 0;
  p.cols = table_cols;
  p.prefix = prefix_len;
  p.causal = causal;
  p.runs = (int)max_runs(table_cols, p.ps, prefix_len);
  p.mtiles = (p.G * p.L + kRows - 1) / kRows;
  p.num_pages = pages->num_pages;
  p.table_stride = table_stride;
  p.scale = scale;
  p.table = page_table;
  p.lens = seq_lens;
  p.prefix_table = prefix_table;
  p.cb = codec->centroids;
  p.perm = codec->permutation;
  p.heavy_mask = p.n_heavy ? codec->heavy_mask : nullptr;
  p.idx = pages->indices;
  p.heavy = pages->heavy;
  p.val = pages->value;
  p.out = out;
  p.part = static_cast<float*>(workspace);
  p.err = paged_error_word();
  if (!p.err) return set_last_error(SUNSHAPE_E_CUDA, "the paged error word is unavailable on this device.");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (pages->dtype == SUNSHAPE_BF16) launch<__nv_bfloat16>(p, st);
  else launch<__half>(p, st);
  return launch_status("paged attention launch");
}

}  // extern "C"
