// Attention of queries over the keys of their own document: capped scores, a bias that
// falls with the distance along up to three position axes, causal order with a prefix
// that every query sees. Documents lie one behind another in the token rows.
//
// Per head h and query i of a document of nq queries and nk keys
//   z_j = scale <q_i, k_j>;  z_j = cap tanh(z_j / cap);
//   z_j -= sum_a |slope[a][h]| |qpos[a][i] - kpos[a][j]|
//   o_i = sum_{j < seen(i)} exp(z_j - m) v_j / sum_{j < seen(i)} exp(z_j - m)
// All masks together leave each query a run of its document's first keys:
//   seen(i) = nk, or with causal order min(nk, max(prefix, i + 1 + nk - nq)).
// Scores, maxima, sums and outputs are fp32 until the one rounding of o. The tile kernels hold
// the scores as the products give them, caps and biases divided by `scale`; scale log2 e comes
// in with the difference to the row's maximum, in front of the exponential, which is one of base 2.
// That difference is made before the product where scores may be large: a rounded product with the
// maximum alone is off by 2^4 and more from scores of 2^28 on, out of the weights' and the sums' range.
#include "heads.cuh"

namespace s2s {
namespace {

struct Rows {
  void* data;
  int64_t token, head;  // strides
};

struct AttnArgs {
  Rows q, k, v, out;
  float* lse;
  const int *qoff, *koff, *prefix;
  const int *qpos, *kpos;
  const float* slopes;
  int q_tokens, kv_tokens, documents, causal, axes;
  int q_heads, kv_heads, group, head_dim;
  int splits;      // CTAs of a cluster that share a tile's keys
  int slots;       // of row tiles (find_document)
  unsigned long long guess;  // documents per slot, 32.32 fixed point
  int cta_heads;   // key heads that a CTA takes, one after the other
  unsigned launch;  // a number of the call's own
  float scale, cap;
};

constexpr int kMaxSplits = 16;  // the largest cluster
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Waits that gave up in these kernels, apart from the library's error word, so that neither side
// stops the other's calls or takes its reports: the first one's code, for s2s_device_status
// alone, and the call that had the last one, whose other waits then do not run out.
struct GaveUp {
  unsigned code, launch;
};
__device__ GaveUp g_attention_gave_up = {0, 0};

__device__ __forceinline__ bool attn_wait(unsigned launch, uint64_t* bar, uint32_t phase, unsigned code,
                                          uint64_t limit_ns = 2000000000ull) {
  return mbar_wait_bounded(
      bar, phase, limit_ns,
      [&] {
        atomicCAS(&g_attention_gave_up.code, 0u, code);
        atomicExch(&g_attention_gave_up.launch, launch);
      },
      [&] { return *(volatile unsigned*)&g_attention_gave_up.launch == launch; });
}

// A wait that nobody meets, for `limit_ns`, recorded as a forward's or as an attention call's.
__global__ void k_wait_gives_up(int attention, unsigned launch, uint64_t limit_ns) {
  __shared__ uint64_t bar;
  mbar_init(&bar, 1);
  fence_barrier_init();
  if (attention)
    attn_wait(launch, &bar, 0, DEV_TIMEOUT_FULL, limit_ns);
  else
    mbar_wait_bounded(&bar, 0, limit_ns, [] { record_error(DEV_TIMEOUT_FULL); }, [] { return false; });
}

// 1, 2, ...
inline unsigned next_launch() {
  static std::atomic<unsigned> last{0};
  unsigned n = ++last;
  while (n == 0) n = ++last;
  return n;
}

struct Doc {
  int q0, nq, k0, nk, prefix;
};

// Offsets are device data that the host cannot check: cut to the tokens, so that no row
// outside the tensors is ever touched.
__device__ __forceinline__ Doc document(const AttnArgs& A, int d) {
  Doc D;
  if (A.qoff) {
    D.q0 = min(max(A.qoff[d], 0), A.q_tokens);
    D.nq = min(max(A.qoff[d + 1], D.q0), A.q_tokens) - D.q0;
    D.k0 = min(max(A.koff[d], 0), A.kv_tokens);
    D.nk = min(max(A.koff[d + 1], D.k0), A.kv_tokens) - D.k0;
  } else {
    D.nq = A.q_tokens / A.documents;
    D.nk = A.kv_tokens / A.documents;
    D.q0 = d * D.nq;
    D.k0 = d * D.nk;
  }
  D.prefix = A.prefix ? A.prefix[d] : 0;
  return D;
}

// Tiles of `rows` rows (`mult` rows a query) lie in `slots` slots: document d's tiles begin at
// slot floor(rows before it / rows) + d, which leaves each document room for all of them
// without a look at the others. The document of a slot, by a whole warp, and the slot's tile
// in it; false where there is none. Documents of about one length are found at the first
// guess, in one round of loads; others by a search of 32 places a round.
__device__ __forceinline__ bool find_document(const AttnArgs& A, int slot, int rows, int mult, int lane,
                                              Doc* D, int* tile) {
  auto first = [&](int d) -> int {
    const int q = A.qoff ? min(max(A.qoff[d], 0), A.q_tokens) : d * (A.q_tokens / A.documents);
    return (int)((unsigned)(q * mult) / (unsigned)rows) + d;  // q_tokens * group is below 2^31
  };
  const int d = min(A.documents - 1, (int)((slot * A.guess) >> 32));
  *D = document(A, d);
  const int at = first(d), next = d + 1 < A.documents ? first(d + 1) : slot + 1;
  if (at <= slot && slot < next) {
    *tile = slot - at;
    return true;
  }
  int lo = 0, n = A.documents;  // the last d of [lo, lo + n) with first(d) <= slot
  while (n > 1) {
    const int step = (n + 31) / 32, x = lo + lane * step;
    const unsigned ok = __ballot_sync(0xffffffffu, lane * step < n && first(x) <= slot);
    const int c = max(__popc(ok) - 1, 0) * step;
    lo += c;
    n = min(step, n - c);
  }
  *D = document(A, lo);
  *tile = slot - first(lo);
  return *tile >= 0;
}

// The slots of a call with tiles of `rows` rows.
inline void set_slots(AttnArgs& A, int rows, int mult) {
  A.slots = (int)((long long)A.q_tokens * mult / rows + A.documents);
  A.guess = (((unsigned long long)A.documents << 32) + A.slots - 1) / A.slots;
}

// Keys that query i of the document sees.
__device__ __forceinline__ int seen(const AttnArgs& A, const Doc& D, int i) {
  if (!A.causal) return D.nk;
  const long long last = (long long)i + 1 + D.nk - D.nq;
  return (int)min((long long)D.nk, max(last, (long long)max(D.prefix, 0)));
}

// The bias of one pair, times log2 e; positions may lie anywhere in 32 bits.
__device__ __forceinline__ float distance_bias(const AttnArgs& A, int h, int qrow, int krow) {
  float b = 0.0f;
  for (int a = 0; a < A.axes; a++) {
    const long long d = (long long)A.qpos[(int64_t)a * A.q_tokens + qrow] -
                        A.kpos[(int64_t)a * A.kv_tokens + krow];
    b -= fabsf(A.slopes[a * A.q_heads + h]) * kLog2e * (float)(d < 0 ? -d : d);
  }
  return b;
}

using F2 = unsigned long long;  // two fp32 lanes of the packed operations
__device__ __forceinline__ F2 f2_both(float x) { return f2_pack(x, x); }
__device__ __forceinline__ F2 f2_abs(F2 x) { return x & 0x7fffffff7fffffffull; }

// log sum exp of a row from its largest score m and the sum l of its weights, which are 2^LIFT times
// exp(z - m).
template <int LIFT>
__device__ __forceinline__ float log_sum(float m, float unit, float l) {
  return fmaf(m, unit, log2f(l * (1.0f / (1 << LIFT)))) * kLn2;
}

// The larger and the smaller of three.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Capped scores, divided by the scale: s -> raw_cap tanh(s to_cap), where raw_cap to_cap = 1. For
// arguments up to 1, tanh x = x (1 + x^2 Q(x^2)) with Q of least relative error of the whole on [0, 1],
// six coefficients (5.7e-8 as they are rounded, by the exchange algorithm and a search of the last bits),
// up to 0.35 three (4.1e-8); with the roundings of its evaluation 1.7e-7. Where x^2 is below 2^-24 that is x
// itself. Beyond 1, 1 - 2 / (1 + e^{2x}). A warp takes the shortest form that is enough for all its scores:
// caps are there for the exception, and the special function unit is busy with the exponentials.
template <int DEGREE>
__device__ __forceinline__ F2 tanh_over_x(F2 u) {
  F2 p;
  if (DEGREE == 6) {
    p = f2_fma(f2_both(0.0010582684772089124f), u, f2_both(-0.006259354762732983f));
    p = f2_fma(p, u, f2_both(0.020359782502055168f));
    p = f2_fma(p, u, f2_both(-0.053498707711696625f));
    p = f2_fma(p, u, f2_both(0.13326406478881836f));
    p = f2_fma(p, u, f2_both(-0.33332985639572144f));
  } else {
    p = f2_fma(f2_both(-0.04914923757314682f), u, f2_both(0.13299839198589325f));
    p = f2_fma(p, u, f2_both(-0.33332663774490356f));
  }
  return f2_fma(p, u, f2_both(1.0f));
}
__device__ __forceinline__ float tanh_far(float x, float near) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2(fabsf(x) * (2.0f * kLog2e))));
  return fabsf(x) > 1.0f ? copysignf(fmaf(-2.0f, r, 1.0f), x) : near;
}
template <int DEGREE, int N>
__device__ __forceinline__ void cap_by(float (&s)[N], float to_cap) {
  const F2 t = f2_both(to_cap);
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    const F2 v = f2_pack(s[j], s[j + 1]), x = f2_mul(v, t);
    const float2 y = f2_unpack(f2_mul(v, tanh_over_x<DEGREE>(f2_mul(x, x))));
    s[j] = y.x;
    s[j + 1] = y.y;
  }
}
template <int N>
__device__ __forceinline__ void capped(float (&s)[N], float to_cap, float raw_cap) {
  float high = -INFINITY, low = INFINITY;
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    high = max3(high, s[j], s[j + 1]);
    low = min3(low, s[j], s[j + 1]);
  }
  const float far = fmaxf(high, -low) * to_cap;
  if (!__any_sync(0xffffffffu, far > 0.35f)) {
    cap_by<3>(s, to_cap);
  } else if (!__any_sync(0xffffffffu, far > 1.0f)) {
    cap_by<6>(s, to_cap);
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const F2 x = f2_mul(f2_pack(s[j], s[j + 1]), f2_both(to_cap));
      const float2 xs = f2_unpack(x), y = f2_unpack(f2_mul(x, tanh_over_x<6>(f2_mul(x, x))));
      s[j] = raw_cap * tanh_far(xs.x, y.x);
      s[j + 1] = raw_cap * tanh_far(xs.y, y.y);
    }
  }
}

// Before a CTA ends after a wait that gave up: the copy on `bar` has landed, or half a second is over.
__device__ __forceinline__ void wait_landed(uint64_t* bar, uint32_t phase) {
  const uint64_t t0 = global_timer_ns();
  while (!mbar_try_wait(smem_u32(bar), phase) && global_timer_ns() - t0 < 500000000ull) {
  }
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const T* t = reinterpret_cast<const T*>(&u);
  return make_float4(to_f32(t[0]), to_f32(t[1]), to_f32(t[2]), to_f32(t[3]));
}

// A row whose outputs came out NaN or infinite, again by one warp: lane l has the values 4l .. 4l + 3
// of the head. The tile kernels multiply the values of keys that a row does not see by zero weights,
// and zero times NaN or infinity is NaN; `end`: the keys that the row's tile went through. Nothing is
// to be done where those values are finite, or where each column that they reach has a NaN among the
// keys that the row does see; only what is left is computed, key after key. The row's sum is right
// as it is.
template <typename T>
__device__ __noinline__ void attend_row(const AttnArgs& A, const Doc D, int i, int h, int end, int lane) {
  const int qrow = D.q0 + i, hk = h / A.group, d = lane * 4;
  const bool mine = d < A.head_dim;
  const T* k = static_cast<const T*>(A.k.data) + (int64_t)D.k0 * A.k.token + (int64_t)hk * A.k.head + d;
  const T* v = static_cast<const T*>(A.v.data) + (int64_t)D.k0 * A.v.token + (int64_t)hk * A.v.head + d;
  const int n = seen(A, D, i);
  float reached[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // NaN: by a hidden NaN or infinity
  if (mine)
    for (int j = n; j < min(end, D.nk); j++) {
      const float4 x = load4(v + (int64_t)j * A.v.token);
      reached[0] = fmaf(x.x, 0.0f, reached[0]);
      reached[1] = fmaf(x.y, 0.0f, reached[1]);
      reached[2] = fmaf(x.z, 0.0f, reached[2]);
      reached[3] = fmaf(x.w, 0.0f, reached[3]);
    }
  bool open = reached[0] != 0.0f || reached[1] != 0.0f || reached[2] != 0.0f || reached[3] != 0.0f;
  for (int j = 0; __any_sync(0xffffffffu, open) && j < n; j++) {
    if (!open) continue;
    const float4 x = load4(v + (int64_t)j * A.v.token);
    if (x.x != x.x) reached[0] = 0.0f;
    if (x.y != x.y) reached[1] = 0.0f;
    if (x.z != x.z) reached[2] = 0.0f;
    if (x.w != x.w) reached[3] = 0.0f;
    open = reached[0] != 0.0f || reached[1] != 0.0f || reached[2] != 0.0f || reached[3] != 0.0f;
  }
  if (!__any_sync(0xffffffffu, open)) return;

  float4 q = make_float4(0, 0, 0, 0), o = q;
  if (mine)
    q = load4(static_cast<const T*>(A.q.data) + (int64_t)qrow * A.q.token + (int64_t)h * A.q.head + d);
  float m = -INFINITY, l = 0.0f;
  for (int j = 0; j < n; j++) {
    float s = 0.0f;
    if (mine) {
      const float4 x = load4(k + (int64_t)j * A.k.token);
      s = q.x * x.x + q.y * x.y + q.z * x.z + q.w * x.w;
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    float z = s * A.scale;
    if (A.cap > 0.0f) z = A.cap * tanhf(z / A.cap);
    z = z * kLog2e + distance_bias(A, h, qrow, D.k0 + j);
    if (z == -INFINITY) continue;
    const float top = fmaxf(m, z), keep = ex2(m - top), p = ex2(z - top);
    m = top;
    l = l * keep + p;
    if (mine) {
      const float4 x = load4(v + (int64_t)j * A.v.token);
      o.x = o.x * keep + p * x.x;
      o.y = o.y * keep + p * x.y;
      o.z = o.z * keep + p * x.z;
      o.w = o.w * keep + p * x.w;
    }
  }
  const float inv = m == -INFINITY ? 0.0f : 1.0f / l;
  if (mine) {
    uint2 u;
    T* t = reinterpret_cast<T*>(&u);
    t[0] = from_f32<T>(o.x * inv);
    t[1] = from_f32<T>(o.y * inv);
    t[2] = from_f32<T>(o.z * inv);
    t[3] = from_f32<T>(o.w * inv);
    *reinterpret_cast<uint2*>(static_cast<T*>(A.out.data) + (int64_t)qrow * A.out.token +
                              (int64_t)h * A.out.head + d) = u;
  }
}

// Rows of heads as a [tokens][heads][head_dim] tensor, in boxes of `rows` tokens, one head and
// `cols` values (32 or 64; zeros beyond head_dim and beyond the tokens), swizzled over the box's
// rows of 64 or 128 bytes.
inline bool make_map_heads(CUtensorMap* map, const Rows& x, bool bf16, int64_t tokens, int heads,
                           int head_dim, int rows, int cols) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)tokens};
  // a stride that is never used still has to be a valid one
  cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? x.head : head_dim) * 2,
                           (cuuint64_t)(tokens > 1 ? x.token : head_dim) * 2};
  cuuint32_t box[3] = {(cuuint32_t)cols, 1, (cuuint32_t)rows};
  cuuint32_t es[3] = {1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, x.data,
            dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace s2s

#include "masked_attention_mma.cuh"
#include "masked_attention_tc.cuh"

namespace s2s {
namespace {

// Which of the two kernels, by what they measured (B200, cycles): a tcgen05 CTA takes 256 queries
// over a key in 22 and 10000 besides, whatever the head; the mma.sync tiles take 0.25, 0.34 or 0.59
// of an SM for each pair of query and key (head_dim up to 32, 64, 128), in as many CTAs as fill the
// device. At eight heads of 64 and 8192 tokens in all, documents of 192: 23 us by mma.sync, 27 by
// tcgen05; of 256: 26 and 22; of 512: 41 and 24. The lengths are on the device, so the costs are those of
// documents of the mean length. Where lengths are mixed the choice can be the slower kernel: 196, 49
// and 100 queries over 6272, 1813 and 900 keys, 16 heads of 128: mma.sync, 71 us of 98; three times 115 over
// 3000: mma.sync, 63 of 36; one image of 4096 with 60 of 16, 12 heads of 64: mma.sync, 189 of 126; 16384 in
// order with 200 of one, eight heads of 128: mma.sync, 2251 of 516. S2S_MASKED_ATTN=mma or tcgen05 in the
// environment (a validation switch, read at every call) takes that one.
template <typename T>
cudaError_t launch_attention(AttnArgs& A, cudaStream_t st) {
  const double queries = (double)A.q_tokens / A.documents, keys = (double)A.kv_tokens / A.documents;
  const double ctas = std::ceil(queries / (2 * kTcTile)) * A.documents * A.q_heads;
  const double tc = std::ceil(ctas / 148) * (keys * 22 + 10000);
  const double pair = A.head_dim <= 32 ? 0.25 : A.head_dim <= 64 ? 0.34 : 0.59;
  const double mma = (double)A.q_tokens * A.q_heads * keys * pair / 148;
  bool large = tc < mma;
  if (const char* e = getenv("S2S_MASKED_ATTN")) large = !strcmp(e, "tcgen05") || (large && strcmp(e, "mma"));
  return A.kv_tokens > 0 && large ? launch_attention_tc<T>(A, st) : launch_attention_mma<T>(A, st);
}

}  // namespace
}  // namespace s2s

extern "C" {

int s2s_masked_attention(const s2s_attention* a, void* stream) {
  using namespace s2s;
  return guarded_call([&] {
    const std::string me = "s2s_masked_attention: ";
    if (!a) fail(S2S_ERR_INVALID, me + "null argument");
    if (a->dtype != S2S_F16 && a->dtype != S2S_BF16)
      fail(S2S_ERR_INVALID, me + "dtype must be S2S_F16 or S2S_BF16");
    if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8)
      fail(S2S_ERR_INVALID, me + "head_dim must be a multiple of 8, at most 128");
    if (a->q_tokens < 0 || a->kv_tokens < 0 || a->documents < 0)
      fail(S2S_ERR_INVALID, me + "tokens and documents must be >= 0");
    if (!a->d_q_offsets != !a->d_kv_offsets)
      fail(S2S_ERR_INVALID, me + "offsets of queries and keys come together");
    if (!a->d_q_offsets && a->documents > 0 &&
        (a->q_tokens % a->documents || a->kv_tokens % a->documents))
      fail(S2S_ERR_INVALID, me + "without offsets the documents must divide the tokens");
    if (a->d_prefix && !a->causal) fail(S2S_ERR_INVALID, me + "a prefix needs causal order");
    if (!(a->scale >= 1e-12f && a->scale <= 1e12f))
      fail(S2S_ERR_INVALID, me + "scale must be between 1e-12 and 1e12");
    if (a->cap != 0.0f && !(a->cap >= 1e-12f && a->cap <= 1e12f))  // cap / scale and its inverse
      fail(S2S_ERR_INVALID, me + "cap must be 0 or between 1e-12 and 1e12");
    if (a->axes < 0 || a->axes > S2S_MAX_AXES)
      fail(S2S_ERR_INVALID, me + "axes must be 0.." + std::to_string(S2S_MAX_AXES));
    check_heads("s2s_masked_attention: q", a->q, a->q_tokens, a->head_dim, a->dtype, 8, false);
    check_heads("s2s_masked_attention: k", a->k, a->kv_tokens, a->head_dim, a->dtype, 8, false);
    check_heads("s2s_masked_attention: v", a->v, a->kv_tokens, a->head_dim, a->dtype, 8, false);
    check_heads("s2s_masked_attention: out", a->out, a->q_tokens, a->head_dim, a->dtype, 8, true);
    if (a->v.heads != a->k.heads || a->out.heads != a->q.heads || a->q.heads % a->k.heads)
      fail(S2S_ERR_INVALID, me + "k and v, and q and out, must have the same heads, q's a "
                                 "multiple of k's");
    if (a->q.heads > 65535) fail(S2S_ERR_INVALID, me + "at most 65535 heads");
    // what is added to a row's or a key's place (a tile at most) has to stay in 32 bits too
    if ((int64_t)a->q_tokens * (a->q.heads / a->k.heads) > 0x7fffff00)
      fail(S2S_ERR_INVALID, me + "q_tokens * (q heads / k heads) must stay below 2^31");
    if (a->kv_tokens > 0x7fffff00)
      fail(S2S_ERR_INVALID, me + "kv_tokens must be 2^31 - 256 at most");
    if (a->documents > 1 << 30) fail(S2S_ERR_INVALID, me + "at most 2^30 documents");
    for (const void* p : {(const void*)a->d_q_offsets, (const void*)a->d_kv_offsets,
                          (const void*)a->d_prefix, (const void*)a->d_slopes,
                          (const void*)a->d_q_pos, (const void*)a->d_kv_pos,
                          (const void*)a->d_lse})
      if ((uintptr_t)p % 4)
        fail(S2S_ERR_INVALID, me + "offsets, prefix, slopes, positions and lse must be 4-byte "
                                   "aligned");
    if (a->q_tokens == 0 || a->documents == 0) return;
    if (a->axes && (!a->d_slopes || !a->d_q_pos || (!a->d_kv_pos && a->kv_tokens)))
      fail(S2S_ERR_INVALID, me + "axes need d_slopes, d_q_pos and d_kv_pos");
    const bool keys = a->kv_tokens > 0;
    const void *o = a->out.data, *sums = a->d_lse;
    if (o == a->q.data || o == sums || (keys && (o == a->k.data || o == a->v.data)) ||
        (sums && (sums == a->q.data || (keys && (sums == a->k.data || sums == a->v.data)))))
      fail(S2S_ERR_INVALID, me + "out and d_lse may not be an input or one another");
    DeviceScope scope({{"s2s_masked_attention: q", a->q.data},
                       {"s2s_masked_attention: k", keys ? a->k.data : nullptr},
                       {"s2s_masked_attention: v", keys ? a->v.data : nullptr},
                       {"s2s_masked_attention: out", a->out.data},
                       {"s2s_masked_attention: d_q_offsets", a->d_q_offsets},
                       {"s2s_masked_attention: d_kv_offsets", a->d_kv_offsets},
                       {"s2s_masked_attention: d_prefix", a->d_prefix},
                       {"s2s_masked_attention: d_slopes", a->axes ? a->d_slopes : nullptr},
                       {"s2s_masked_attention: d_q_pos", a->axes ? a->d_q_pos : nullptr},
                       {"s2s_masked_attention: d_kv_pos", a->axes && keys ? a->d_kv_pos : nullptr},
                       {"s2s_masked_attention: d_lse", a->d_lse}}, stream);
    AttnArgs A;
    memset(&A, 0, sizeof A);
    auto rows = [](const s2s_heads& x, int64_t tokens) {
      const s2s_heads p = plain_strides(x, tokens);
      return Rows{p.data, p.token_stride, p.head_stride};
    };
    A.q = rows(a->q, a->q_tokens);
    A.k = rows(a->k, a->kv_tokens);
    A.v = rows(a->v, a->kv_tokens);
    A.out = rows(a->out, a->q_tokens);
    A.lse = a->d_lse;
    A.qoff = a->d_q_offsets;
    A.koff = a->d_kv_offsets;
    A.prefix = a->d_prefix;
    A.axes = a->axes;
    A.qpos = a->d_q_pos;
    A.kpos = a->d_kv_pos;
    A.slopes = a->d_slopes;
    A.q_tokens = a->q_tokens;
    A.kv_tokens = a->kv_tokens;
    A.documents = a->documents;
    A.causal = a->causal != 0;
    A.q_heads = a->q.heads;
    A.kv_heads = a->k.heads;
    A.group = a->q.heads / a->k.heads;
    A.head_dim = a->head_dim;
    A.scale = a->scale;
    A.cap = a->cap;
    A.launch = next_launch();
    cudaStream_t st = (cudaStream_t)stream;
    ck(a->dtype == S2S_F16 ? launch_attention<__half>(A, st) : launch_attention<__nv_bfloat16>(A, st),
       "masked_attention");
  });
}

int s2s_debug_attention_loads(int tiles, int waits, int* copies) {
  using namespace s2s;
  return guarded_call([&] {
    if (tiles < 0 || !copies) fail(S2S_ERR_INVALID, "s2s_debug_attention_loads: null argument");
    memset(copies, 0, 2 * (size_t)tiles * sizeof(int));
    constexpr int ST = TcCfg<1>::STAGES;
    load_tiles<ST>(
        tiles,
        [&](bool value, int i) {
          if (waits-- <= 0) return false;
          copies[2 * (i - ST) + value] = 2;
          return true;
        },
        [&](bool value, int i) { copies[2 * i + value] = 1; },
        [&](bool value, int i) { copies[2 * i + value] += 2; });
  });
}

int s2s_device_status(int device) {
  using namespace s2s;
  return guarded_call([&] {
    int before = 0;
    ck(cudaGetDevice(&before), "cudaGetDevice");
    struct Restore {
      int d;
      ~Restore() { cudaSetDevice(d); }
    } restore{before};
    ck(cudaSetDevice(device), "cudaSetDevice");
    ck(cudaDeviceSynchronize(), "cudaDeviceSynchronize");
    GaveUp e, none = {0, 0};
    ck(cudaMemcpyFromSymbol(&e, g_attention_gave_up, sizeof e), "error word");
    if (e.code != 0) {
      ck(cudaMemcpyToSymbol(g_attention_gave_up, &none, sizeof none), "error word");
      fail(S2S_ERR_TIMEOUT, "a wait of an attention call gave up (code " + std::to_string(e.code) +
                                "); its outputs are undefined");
    }
    unsigned forward = 0;  // the next synchronous forward reports and clears it
    ck(cudaMemcpyFromSymbol(&forward, g_s2s_err, sizeof forward), "error word");
    if (forward != 0)
      fail(S2S_ERR_TIMEOUT, "a wait of a forward gave up (code " + std::to_string(forward) +
                                "), which no synchronous forward has reported yet");
  });
}

int s2s_debug_wait_gives_up(int device, int attention) {
  using namespace s2s;
  return guarded_call([&] {
    int before = 0;
    ck(cudaGetDevice(&before), "cudaGetDevice");
    struct Restore {
      int d;
      ~Restore() { cudaSetDevice(d); }
    } restore{before};
    ck(cudaSetDevice(device), "cudaSetDevice");
    k_wait_gives_up<<<1, 1>>>(attention, next_launch(), 20000000ull);
    ck(cudaGetLastError(), "wait_gives_up");
    ck(cudaDeviceSynchronize(), "wait_gives_up");
  });
}

}  // extern "C"
