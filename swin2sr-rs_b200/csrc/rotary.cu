// Rotary positions over several axes: pair p of every head of token t turns by
// position[axis[p]][t] * frequency[p].
//
//   y_a = a cos t - b sin t,   y_b = a sin t + b cos t
//
// Bound: HBM. Every value is read once and written once; the angles of a token are the
// same in all its heads, so a CTA takes up to 16 tokens, makes the (cos, sin) of their
// pairs once into shared memory and then walks the heads of all tensors of the call.
// The turn count position * frequency / 2 pi is reduced to its fraction in 64 bits: at
// position 1e6 a 32-bit product is off by 0.06 rad, this one by less than 1e-9. Sine and
// cosine of the fraction, products and sums are 32-bit.
//
// Measured (B200): 50176 tokens of 16 + 4 heads of 128, bf16: 97 us, 5.3 TB/s (0.81 of the
// measured copy; 90 us where a replay finds a part of its inputs in L2); 81344 tokens of 6 + 6
// heads of 32, fp16: 28 us, 4.5 TB/s. Fewer tokens a CTA
// (8: 33 us at 12 heads of 32) repeat the set-up, two or four loads ahead of the angles take
// the registers that the eight CTAs of an SM need (147 us instead of 90).
#include "heads.cuh"

namespace s2s {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryTokens = 16;  // most tokens of a CTA: 16 x 128 pairs x 8 B = 16 KB
constexpr int kRotaryTensors = 4;

struct RotaryTensor {
  const void* x;
  void* y;
  int64_t xt, xh, yt, yh;  // strides
  int heads;
};

struct RotaryArgs {
  RotaryTensor t[kRotaryTensors];
  int n, heads;  // tensors, heads of all of them
  int axes, pairs, tokens, per_cta, head_dim, inverse;
  const int* pos;
  int64_t pos_stride;
  double turns[S2S_ROTARY_MAX_PAIRS];  // frequency / 2 pi
  uint8_t axis[S2S_ROTARY_MAX_PAIRS];
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

// VEC values per access: 16 bytes where bases, strides and pairs allow it, else one.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads) k_rotary(const __grid_constant__ RotaryArgs A) {
  __shared__ float2 cs[kRotaryTokens * S2S_ROTARY_MAX_PAIRS];
  pdl_trigger();
  const int t0 = blockIdx.x * A.per_cta;
  const int nt = min(A.per_cta, A.tokens - t0);
  pdl_wait();
  // angles: a thread keeps one pair, so its frequency is read once
  const int width = A.pairs <= 32 ? 32 : A.pairs <= 64 ? 64 : 128;
  const int p = threadIdx.x % width;
  if (p < A.pairs) {
    const double f = A.turns[p];
    const int* pos = A.pos + (int64_t)A.axis[p] * A.pos_stride + t0;
    for (int t = threadIdx.x / width; t < nt; t += kRotaryThreads / width) {
      const double turn = (double)pos[t] * f;
      float s, c;
      sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);
      cs[t * A.pairs + p] = make_float2(c, A.inverse ? -s : s);
    }
  }
  __syncthreads();

  // units: one vector of each half's pairs (or VEC / 2 neighbouring pairs), then the
  // values behind the pairs
  const int rot = INTERLEAVED ? 2 * A.pairs / VEC : A.pairs / VEC;
  const int units = rot + (A.head_dim - 2 * A.pairs) / VEC;
  const int total = nt * A.heads * units;
  using V = Vec<T, VEC>;
  for (int u = threadIdx.x; u < total; u += kRotaryThreads) {
    const int row = u / units, k = u - row * units;
    const int t = row / A.heads;
    int h = row - t * A.heads, i = 0;
    while (i + 1 < A.n && h >= A.t[i].heads) h -= A.t[i++].heads;
    const RotaryTensor& R = A.t[i];
    const T* x = static_cast<const T*>(R.x) + (int64_t)(t0 + t) * R.xt + (int64_t)h * R.xh;
    T* y = static_cast<T*>(R.y) + (int64_t)(t0 + t) * R.yt + (int64_t)h * R.yh;
    if (k >= rot) {
      const int d = 2 * A.pairs + (k - rot) * VEC;
      *reinterpret_cast<V*>(y + d) = *reinterpret_cast<const V*>(x + d);
      continue;
    }
    if constexpr (INTERLEAVED) {
      if constexpr (VEC > 1) {
        V v = *reinterpret_cast<const V*>(x + k * VEC);
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
          const float2 r = cs[t * A.pairs + (k * VEC + e) / 2];
          const float a = to_f32(v.v[e]), b = to_f32(v.v[e + 1]);
          v.v[e] = from_f32<T>(a * r.x - b * r.y);
          v.v[e + 1] = from_f32<T>(a * r.y + b * r.x);
        }
        *reinterpret_cast<V*>(y + k * VEC) = v;
      } else if ((k & 1) == 0) {  // one thread has the pair: x may be y
        const float2 r = cs[t * A.pairs + k / 2];
        const float a = to_f32(x[k]), b = to_f32(x[k + 1]);
        y[k] = from_f32<T>(a * r.x - b * r.y);
        y[k + 1] = from_f32<T>(a * r.y + b * r.x);
      }
    } else {
      V va = *reinterpret_cast<const V*>(x + k * VEC);
      V vb = *reinterpret_cast<const V*>(x + A.pairs + k * VEC);
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        const float2 r = cs[t * A.pairs + k * VEC + e];
        const float a = to_f32(va.v[e]), b = to_f32(vb.v[e]);
        va.v[e] = from_f32<T>(a * r.x - b * r.y);
        vb.v[e] = from_f32<T>(a * r.y + b * r.x);
      }
      *reinterpret_cast<V*>(y + k * VEC) = va;
      *reinterpret_cast<V*>(y + A.pairs + k * VEC) = vb;
    }
  }
}

template <typename T, int VEC>
cudaError_t launch_rotary(const RotaryArgs& A, bool interleaved, cudaStream_t st) {
  // in 64 bits: tokens go up to 2^31 - 1
  const dim3 grid((unsigned)(((long long)A.tokens + A.per_cta - 1) / A.per_cta)), block(kRotaryThreads);
  return interleaved ? launch_pdl(k_rotary<T, VEC, true>, grid, block, 0, st, A)
                     : launch_pdl(k_rotary<T, VEC, false>, grid, block, 0, st, A);
}

template <typename T>
cudaError_t launch_rotary(const RotaryArgs& A, bool interleaved, bool wide, cudaStream_t st) {
  return wide ? launch_rotary<T, 16 / (int)sizeof(T)>(A, interleaved, st)
              : launch_rotary<T, 1>(A, interleaved, st);
}

}  // namespace
}  // namespace s2s

extern "C" {

int s2s_rotary_init(s2s_rotary* r, int axes, const int* sections, double base, int per_axis,
                    int interleaved) {
  using namespace s2s;
  return guarded_free([&] {
    if (!r || !sections) fail(S2S_ERR_INVALID, "s2s_rotary_init: null argument");
    if (axes < 1 || axes > S2S_MAX_AXES)
      fail(S2S_ERR_INVALID, "s2s_rotary_init: axes must be 1.." + std::to_string(S2S_MAX_AXES));
    if (!(base > 0.0) || !std::isfinite(base))
      fail(S2S_ERR_INVALID, "s2s_rotary_init: base must be positive and finite");
    int pairs = 0;
    for (int a = 0; a < axes; a++) {
      if (sections[a] < 0 || sections[a] > S2S_ROTARY_MAX_PAIRS)
        fail(S2S_ERR_INVALID, "s2s_rotary_init: a section must be 0.." +
                                  std::to_string(S2S_ROTARY_MAX_PAIRS) + " pairs");
      pairs += sections[a];
    }
    if (pairs < 1 || pairs > S2S_ROTARY_MAX_PAIRS)
      fail(S2S_ERR_INVALID, "s2s_rotary_init: the sections must sum to 1.." +
                                std::to_string(S2S_ROTARY_MAX_PAIRS) + " pairs");
    s2s_rotary out;
    memset(&out, 0, sizeof out);
    out.axes = axes;
    out.pairs = pairs;
    out.interleaved = interleaved != 0;
    int p = 0;
    for (int a = 0; a < axes; a++)
      for (int i = 0; i < sections[a]; i++, p++) {
        out.axis[p] = (uint8_t)a;
        out.frequency[p] = per_axis ? std::pow(base, -(double)i / sections[a])
                                    : std::pow(base, -(double)p / pairs);
      }
    *r = out;
  });
}

int s2s_rotary_apply(const s2s_rotary* r, int dtype, int head_dim, int tokens, const int* d_pos,
                     int64_t pos_stride, const s2s_heads* x, const s2s_heads* y, int n,
                     int inverse, void* stream) {
  using namespace s2s;
  return guarded_call([&] {
    const std::string me = "s2s_rotary_apply: ";
    if (!r || !x || !y) fail(S2S_ERR_INVALID, me + "null argument");
    if (dtype != S2S_F16 && dtype != S2S_BF16 && dtype != S2S_F32)
      fail(S2S_ERR_INVALID, me + "dtype must be S2S_F16, S2S_BF16 or S2S_F32");
    if (r->axes < 1 || r->axes > S2S_MAX_AXES || r->pairs < 1 || r->pairs > S2S_ROTARY_MAX_PAIRS)
      fail(S2S_ERR_INVALID, me + "axes or pairs out of range");
    if (head_dim < 2 * r->pairs || head_dim > 65536)
      fail(S2S_ERR_INVALID, me + "head_dim must be 2 * pairs or more");
    if (tokens < 0) fail(S2S_ERR_INVALID, me + "tokens must be >= 0");
    if (n < 1 || n > kRotaryTensors) fail(S2S_ERR_INVALID, me + "n must be 1..4");
    RotaryArgs A;
    memset(&A, 0, sizeof A);
    for (int p = 0; p < r->pairs; p++) {
      if (r->axis[p] >= r->axes) fail(S2S_ERR_INVALID, me + "a pair's axis is out of range");
      if (!std::isfinite(r->frequency[p]))
        fail(S2S_ERR_INVALID, me + "a pair's frequency is not finite");
      A.axis[p] = r->axis[p];
      A.turns[p] = r->frequency[p] * 0.15915494309189533577;  // 1 / (2 pi)
    }
    const int eb = element_bytes(dtype), vec = 16 / eb;
    bool wide = head_dim % vec == 0 && (2 * r->pairs) % vec == 0 &&
                (r->interleaved || r->pairs % vec == 0);
    long long heads = 0;
    for (int i = 0; i < n; i++) {
      check_heads("s2s_rotary_apply: x", x[i], tokens, head_dim, dtype, 1, false);
      check_heads("s2s_rotary_apply: y", y[i], tokens, head_dim, dtype, 1, true);
      if (x[i].heads != y[i].heads) fail(S2S_ERR_INVALID, me + "x and y differ in heads");
      const s2s_heads a = plain_strides(x[i], tokens), b = plain_strides(y[i], tokens);
      A.t[i] = {a.data, b.data, a.token_stride, a.head_stride, b.token_stride, b.head_stride,
                a.heads};
      for (const s2s_heads& v : {a, b})
        wide = wide && (uintptr_t)v.data % 16 == 0 && v.token_stride % vec == 0 &&
               v.head_stride % vec == 0;
      heads += a.heads;
    }
    if (tokens > 0)
      for (int i = 0; i < n; i++)
        for (int j = 0; j < n; j++) {
          const RotaryTensor &a = A.t[i], &b = A.t[j];
          if (i != j && (a.y == b.y || a.y == b.x))
            fail(S2S_ERR_INVALID, me + "an output is another tensor of the call");
          if (i == j && a.y == a.x && (a.yt != a.xt || a.yh != a.xh))
            fail(S2S_ERR_INVALID, me + "in place, x and y must have the same strides");
        }
    if (heads * head_dim > (1 << 26)) fail(S2S_ERR_INVALID, me + "too many heads");
    if (tokens == 0) return;
    if (!d_pos || (uintptr_t)d_pos % 4) fail(S2S_ERR_INVALID, me + "d_pos must be 4-byte aligned");
    if (r->axes > 1 && pos_stride < tokens)
      fail(S2S_ERR_INVALID, me + "pos_stride is less than tokens");
    DeviceScope scope({{"s2s_rotary_apply: x[0]", x[0].data}, {"s2s_rotary_apply: y[0]", y[0].data},
                       {"s2s_rotary_apply: x[1]", n > 1 ? x[1].data : nullptr},
                       {"s2s_rotary_apply: y[1]", n > 1 ? y[1].data : nullptr},
                       {"s2s_rotary_apply: x[2]", n > 2 ? x[2].data : nullptr},
                       {"s2s_rotary_apply: y[2]", n > 2 ? y[2].data : nullptr},
                       {"s2s_rotary_apply: x[3]", n > 3 ? x[3].data : nullptr},
                       {"s2s_rotary_apply: y[3]", n > 3 ? y[3].data : nullptr},
                       {"s2s_rotary_apply: d_pos", d_pos}}, stream);
    A.n = n;
    A.heads = (int)heads;
    A.axes = r->axes;
    A.pairs = r->pairs;
    A.tokens = tokens;
    A.head_dim = head_dim;
    A.inverse = inverse != 0;
    A.pos = d_pos;
    A.pos_stride = r->axes > 1 ? pos_stride : 0;
    // few tokens: one per CTA, so that the call spreads over the SMs
    A.per_cta = std::max(1, std::min(kRotaryTokens, tokens / (148 * 8)));
    const bool il = r->interleaved != 0;
    cudaStream_t st = (cudaStream_t)stream;
    ck(dtype == S2S_F16    ? launch_rotary<__half>(A, il, wide, st)
       : dtype == S2S_BF16 ? launch_rotary<__nv_bfloat16>(A, il, wide, st)
                           : launch_rotary<float>(A, il, wide, st),
       "rotary");
  });
}

}  // extern "C"
