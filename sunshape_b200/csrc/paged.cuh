// Arguments and helpers shared by the paged-serving kernels (norm_rotate.cu, paged_append.cu,
// paged_attention.cu).
#pragma once

#include <atomic>

#include "common.cuh"

namespace sunshape {

enum PagedError { kErrPosition = 131, kErrSlot = 132, kErrPage = 133, kErrLength = 134, kErrWait = 135, kErrDense = 136 };

// device address of the paged kernels' error word on the current device (null with a CUDA error set)
int* paged_error_word();
// reports through sunshape_last_error(), capi.cu
int set_last_error(int code, const char* msg);
// the status of the launches just made, capi.cu
int launch_status(const char* what);
// argument checks shared with the contiguous entry points, capi.cu
int check_codec_args(const sunshape_codec_t* c);
// SMs of the current device, capi.cu; and the same, asked once a device
int sm_count();
int paged_sm_count();
// Lets a kernel use `smem` bytes of dynamic shared memory -- the most that any call of it asks for -- and checks that it
// was built for `regs` registers (0: any number), once a device.
bool ready_kernel(const void* kernel, int smem, int regs, std::atomic<uint64_t>& done);
// checks a page pool against its codec, paged_append.cu
int check_pages(const sunshape_codec_t* c, const sunshape_pages_t* pg);

// What the paged kernels read of a codec, in one buffer (paged_append.cu fills it).
//   image   at 0, [n_cb][ceil(D / 64)][256][64] fp16: codewords times their codebook's image scale; row (i, c) holds codeword
//           c of the 64 / BD blocks from i * 64 / BD on, so that in shared memory a block's codewords lie in one
//           column of the banks
//   iscale  [n_cb]: the image's scale, a power of two that brings the codebook's largest codeword norm into [0.5, 1), at most 1
//           where the codec has dense blocks
//   records [n_cb][nb]: what the encoder reads of a block, one copy each --
//     frags [32][32][2]: the B operands of the MMAs over 8 codewords, lane by lane
//     norms [256]: -|c|^2 / 2 in the block's scale, far below all others where there is no codeword
//     words [256][BD] fp32, far from all others where there is no codeword
//     scale: a power of two that brings the block's largest codeword norm into [0.5, 1); three unused
constexpr int kRecNorms = 8192, kRecWords = 9216;
__host__ __device__ constexpr int record_bytes(int bd) { return kRecWords + 1024 * bd + 16; }

struct Tables {
  int64_t iscale, records, total;
  __host__ __device__ Tables(int64_t n_cb, int64_t nb, int64_t D) {
    iscale = n_cb * ((D + 63) / 64) * 32768;
    records = iscale + (n_cb * 4 + 255) / 256 * 256;
    total = records + (n_cb * nb * record_bytes((int)(D / nb)) + 255) / 256 * 256;
  }
};

// Rotation arguments as the kernels take them; rot = 0 without a rotation.
struct Rotation {
  const float* cos;
  const float* sin;
  const void* pos;
  int64_t pos_sb, pos_sl, table_len;
  int pos64, rot, interleaved;
};

// checks a rotation; `empty`: the call has no rows and its pointers may be null
int make_rotation(const sunshape_rotation_t* r, int dim, bool empty, Rotation* out);

// position of token (b, l); the caller checks the table's range
__device__ __forceinline__ int64_t position_of(const Rotation& r, int64_t b, int64_t l) {
  const int64_t i = b * r.pos_sb + l * r.pos_sl;
  return r.pos64 ? reinterpret_cast<const int64_t*>(r.pos)[i] : (int64_t) reinterpret_cast<const int32_t*>(r.pos)[i];
}

// the other element of element d's pair, the pair's index, and whether d is the second of the two (d < rot)
__device__ __forceinline__ void pair_of(const Rotation& r, int d, int& other, int& i, bool& second) {
  if (r.interleaved) {
    other = d ^ 1;
    i = d >> 1;
    second = d & 1;
  } else {
    const int half = r.rot >> 1;
    second = d >= half;
    other = second ? d - half : d + half;
    i = second ? d - half : d;
  }
}

template <typename T> struct Elem;
template <> struct Elem<float> {
  static __device__ __forceinline__ float to_float(float v) { return v; }
  static __device__ __forceinline__ float from_float(float v) { return v; }
};
template <> struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Elem<__half> {
  static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
};

}  // namespace sunshape
