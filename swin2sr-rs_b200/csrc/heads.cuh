// Host-side checks and launch scope shared by the token operators (rotary.cu,
// masked_attention.cu): element types, rows of heads, and the device the tensors live on.
#pragma once
#include <cuda_bf16.h>

namespace s2s {
namespace {

inline int element_bytes(int dtype) { return dtype == S2S_F32 ? 4 : 2; }

// `x` as `tokens` rows of heads of `head_dim` values, each row starting on a multiple of
// `align` elements. Rows that are written (`out`) must not run into one another.
void check_heads(const char* what, const s2s_heads& x, int64_t tokens, int head_dim, int dtype,
                 int align, bool out) {
  const std::string w = what;
  if (x.heads < 1) fail(S2S_ERR_INVALID, w + ": heads must be >= 1");
  if (tokens == 0) return;
  if (!x.data) fail(S2S_ERR_INVALID, w + ": null data");
  if ((uintptr_t)x.data % ((size_t)align * element_bytes(dtype)))
    fail(S2S_ERR_INVALID, w + ": data must be " + std::to_string(align * element_bytes(dtype)) +
                              "-byte aligned");
  const int64_t most = (int64_t)1 << 38;  // of a stride, in elements
  auto stride = [&](const char* name, int64_t s) {
    if (s < 1 || s > most || s % align)
      fail(S2S_ERR_INVALID, w + ": " + name + " must be positive" +
                                (align > 1 ? " and a multiple of " + std::to_string(align) : ""));
    if (out && s < head_dim) fail(S2S_ERR_INVALID, w + ": " + name + " is less than head_dim");
  };
  if (tokens > 1) stride("token_stride", x.token_stride);
  if (x.heads > 1) stride("head_stride", x.head_stride);
  if (out && tokens > 1 && x.heads > 1) {
    const bool inner = x.head_stride <= x.token_stride;  // the heads lie within a token's row
    const int64_t small = inner ? x.head_stride : x.token_stride, n = inner ? x.heads : tokens;
    const int64_t large = inner ? x.token_stride : x.head_stride;
    if ((double)small * (n - 1) + head_dim > (double)large)
      fail(S2S_ERR_INVALID, w + ": its rows run into one another");
  }
  // the last element's offset has to be a 64-bit number of bytes with room to spare
  const double last = (double)(tokens - 1) * (double)(tokens > 1 ? x.token_stride : 0) +
                      (double)(x.heads - 1) * (double)(x.heads > 1 ? x.head_stride : 0) + head_dim;
  if (last > 1e18) fail(S2S_ERR_INVALID, w + ": the tensor is too large");
}

// Strides that are never multiplied by anything but zero may hold anything: make them plain.
s2s_heads plain_strides(s2s_heads x, int64_t tokens) {
  if (tokens <= 1) x.token_stride = 0;
  if (x.heads <= 1) x.head_stride = 0;
  return x;
}

// guarded_free for calls that leave no CUDA error behind: one that is reported here would else be
// found by the next look at the runtime's last error, another library's included.
template <typename F>
int guarded_call(F&& f) {
  const int rc = guarded_free(f);
  if (rc == S2S_ERR_CUDA) cudaGetLastError();
  return rc;
}

// For the lifetime of the object the device that holds the tensors is the current one.
// Every pointer has to be memory of that device, the stream one of its streams.
class DeviceScope {
 public:
  DeviceScope(std::initializer_list<std::pair<const char*, const void*>> tensors, void* stream) {
    int dev = -1;
    for (const auto& t : tensors) {
      if (!t.second) continue;
      cudaPointerAttributes at;
      ck(cudaPointerGetAttributes(&at, t.second), "cudaPointerGetAttributes");
      if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
        fail(S2S_ERR_INVALID, std::string(t.first) + " is not device memory");
      if (at.type == cudaMemoryTypeManaged) continue;
      if (dev >= 0 && at.device != dev)
        fail(S2S_ERR_INVALID, std::string(t.first) + " is on device " + std::to_string(at.device) +
                                  ", other tensors are on device " + std::to_string(dev));
      dev = at.device;
    }
    ck(cudaGetDevice(&before_), "cudaGetDevice");
    if (dev < 0) dev = before_;
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (stream && stream != cudaStreamLegacy && stream != cudaStreamPerThread)
      ck(cudaStreamIsCapturing((cudaStream_t)stream, &capture), "cudaStreamIsCapturing");
    else
      stream = nullptr;  // the current device's own
    if (stream && capture == cudaStreamCaptureStatusNone) {  // a capturing stream cannot be asked
      int sdev = -1;
      ck(cudaStreamGetDevice((cudaStream_t)stream, &sdev), "cudaStreamGetDevice");
      if (sdev != dev)
        fail(S2S_ERR_INVALID, "the stream is of device " + std::to_string(sdev) +
                                  ", the tensors are on device " + std::to_string(dev));
    }
    if (dev != before_) {
      ck(cudaSetDevice(dev), "cudaSetDevice");
      changed_ = true;
    }
  }
  ~DeviceScope() {
    if (changed_) cudaSetDevice(before_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;

 private:
  int before_ = 0;
  bool changed_ = false;
};

// ------------------------------------------------------------------ element types
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

}  // namespace
}  // namespace s2s
