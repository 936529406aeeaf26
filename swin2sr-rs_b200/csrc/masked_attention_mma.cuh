// The attention of masked_attention.cu on mma.sync tiles, for short documents, few queries
// and small work.
//
// A CTA of four warps (eight where it has an SM for itself) takes 16 * RW rows of one document and
// key head - a row is a query and one of the query heads that share the key head, so K and V are
// read once for all of them - and walks the keys in tiles of 16 a warp through a ring of three
// stages that TMA fills. RW warps lie along the rows, the others along the keys of a tile: one
// query of eight heads is one row tile, whose keys the warps share. Every warp keeps a running
// maximum, sum and output of its own; they are joined once at the end, first within the CTA, then over
// the CTAs of a cluster among which the keys of the tile were split (through distributed shared memory:
// a call needs no workspace, and the order of the sums is fixed).
//
// Bound: HBM where the keys are long (K and V are read once), else the latency of a tile's chain of
// products, softmax and products, of which an SM has eight to sixteen warps' worth to hide. Measured
// (B200): 24 single queries of 32 heads over 111 000 keys of 8 x 128, 444 MB: 102 us, 4.3 TB/s
// (68 us at the measured copy rate); 1271 windows of 64, six heads of 32, two axes: 55 us (45
// without a bias, 19 for the bytes; issue slots 0.43, no unit above 0.3); 5 queries of 16 heads over
// 40001 keys of 2 x 128: 29 us.
#pragma once

namespace s2s {
namespace {

constexpr int kMmaStages = 3;

// Weights are at most 2^kMmaLift: in fp16, whose least value is 2^-24, those down to 2^-39 of the largest
// then count in the second product. (At most 1, the 65535 keys that share 0.2 % of a row's sum at 2^-25
// each were lost.)
template <typename T>
constexpr int kMmaLift = std::is_same<T, __half>::value ? 15 : 0;

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) { return pack_h2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T>
__device__ __forceinline__ void mma_tile(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma_tile<__half>(float (&c)[4], const uint32_t (&a)[4],
                                                 uint32_t b0, uint32_t b1) {
  mma16816(c, a[0], a[1], a[2], a[3], b0, b1);
}
template <>
__device__ __forceinline__ void mma_tile<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4],
                                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same onto zeros.
template <typename T>
__device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// ------------------------------------------------------------------------- clusters
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ float cluster_load(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\t"
      "ld.shared::cluster.f32 %0, [a];\n\t}"
      : "=f"(v)
      : "r"(addr), "r"(rank));
  return v;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [a];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(addr), "r"(rank));
  return v;
}

template <int DP, int RW, int WARPS, int NA = S2S_MAX_AXES>
struct MmaCfg {
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int TKEYS = 16 * WARPS;       // keys of a tile
  static constexpr int KW = WARPS / RW;          // warps along the keys
  static constexpr int ROWS = 16 * RW;
  static constexpr int KEYS = TKEYS / KW;        // keys of a tile that one warp takes
  static constexpr int PV = DP < 64 ? DP : 64;   // values of a panel: a TMA box's row
  static constexpr int PANEL = TKEYS * PV * 2;
  static constexpr int TILE = TKEYS * DP * 2;    // bytes of a K or V tile, panel after panel
  static constexpr int RING = kMmaStages * 2 * TILE;
  static constexpr int LD = DP + 4;              // floats of a joined output row
  static constexpr int JOIN = WARPS * 16 * LD * 4;  // the warps' outputs, over the ring
  static constexpr int BODY = RING > JOIN ? RING : JOIN;
  static constexpr int POS = S2S_MAX_AXES * TKEYS * 4;  // key positions of a stage
  static constexpr int BARS = BODY + kMmaStages * POS;
  static constexpr int ENDS = BARS + kMmaStages * 8 + 8;   // maxima and sums, flags
  static constexpr int SMEM = ENDS + WARPS * 16 * 8 + ROWS * 12 + 1024;  // + alignment
  // Resident CTAs that the registers are cut to: the more, the more loads are in flight, but what
  // spills costs more (1271 windows of 64, six heads of 32, two axes: 3 CTAs 55 us, 4 67 us; 32
  // single queries over 3000 keys, eight heads of 64: 4 CTAs 44 us, 3 49 us).
  static constexpr int CTAS = (RW < 4   ? (DP == 128 ? 2 : 4)
                               : DP == 32 ? 3
                               : DP == 64 ? (NA ? 2 : 3)
                                          : 2) * 4 / WARPS;
};

// Where lane `lane` finds, in a tile, chunk `b` (16 bytes) of row `r`; chunk b + 2k of the same
// panel is at this offset ^ (32 k), as the swizzle permutes the chunks of a row by exclusive or.
template <int DP>
__device__ __forceinline__ uint32_t tile_at(int r, int b) {
  return DP == 32 ? (uint32_t)(r * 64 + ((b ^ ((r >> 1) & 3)) << 4))
                  : (uint32_t)(r * 128 + ((b ^ (r & 7)) << 4));
}

// Outputs of a head from the warps that have their rows to themselves; `op`: this lane's place in
// its two rows. Whether one of them is NaN or infinite (in causal order, where it matters).
template <typename T, int DN>
__device__ __forceinline__ bool write_rows(const AttnArgs& A, int hk, const float (&o)[DN][4],
                                           const float (&m)[2], const float (&l)[2], float unit, T* const (&op)[2],
                                           const int (&row_q)[2], const int (&row_h)[2],
                                           const bool (&live)[2], int lane) {
  float check = 0.0f;
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const bool none = m[e] == -INFINITY && l[e] == 0.0f;  // a sum that is NaN is kept
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(l[e]));
    if (none) inv = 0.0f;
    if (live[e]) {
#pragma unroll
      for (int n = 0; n < DN; n++)
        if (n * 8 < A.head_dim)
          *reinterpret_cast<uint32_t*>(op[e] + n * 8) = pack2<T>(o[n][2 * e] * inv, o[n][2 * e + 1] * inv);
      if ((lane & 3) == 0 && A.lse)
        A.lse[(int64_t)(hk * A.group + row_h[e]) * A.q_tokens + row_q[e]] =
            none ? -INFINITY : log_sum<kMmaLift<T>>(m[e], unit, l[e]);
    }
    if (A.causal)
#pragma unroll
      for (int n = 0; n < DN; n++) check = fmaf(o[n][2 * e] * inv, 0.0f, fmaf(o[n][2 * e + 1] * inv, 0.0f, check));
  }
  return check != 0.0f;  // true for NaN
}

// Keys that a row does not see are multiplied by zero weights: a NaN or infinity among their values
// shows in the row's outputs. Such rows of this warp are done again without those keys; `op` as it
// was for the first head. Behind the heads' loop, as a call in it costs registers there.
template <typename T, int DN>
__device__ __forceinline__ void mend_rows(const AttnArgs& A, const Doc& D, int hk0, int hk1, T* (&op)[2],
                                          const int (&row_q)[2], const int (&row_h)[2],
                                          const int (&row_seen)[2], const bool (&live)[2], int kend, int lane) {
  for (int hk = hk0; hk < hk1; hk++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      float check = 0.0f;
      if (live[e] && row_seen[e] < kend)
        for (int n = 0; n * 8 < A.head_dim; n++) {
          const uint32_t u = *reinterpret_cast<const uint32_t*>(op[e] + n * 8);
          const T* x = reinterpret_cast<const T*>(&u);
          check = fmaf(to_f32(x[0]), 0.0f, fmaf(to_f32(x[1]), 0.0f, check));
        }
      op[e] += (int64_t)A.group * A.out.head;
      unsigned redo = __ballot_sync(0xffffffffu, check != 0.0f);
      while (redo) {
        const int src = __ffs(redo) - 1;
        redo &= ~(15u << (src & ~3));
        const int i = __shfl_sync(0xffffffffu, row_q[e], src) - D.q0;
        attend_row<T>(A, D, i, hk * A.group + __shfl_sync(0xffffffffu, row_h[e], src), kend, lane);
      }
    }
}

// Outputs of a head whose keys lie with several warps, and CTAs of a cluster: everything they
// have goes through shared memory (over the ring, which is idle by then).
template <typename T, int DP, int RW, int WARPS>
__device__ __forceinline__ void join_rows(const AttnArgs& A, const Doc& D, int hk, uint8_t* smem,
                                          const float (&o)[DP / 8][4], const float (&m)[2],
                                          const float (&l)[2], float unit, int r0, int nrows, int kend,
                                          int S, int split) {
  using C = MmaCfg<DP, RW, WARPS>;
  constexpr int KW = C::KW, DN = DP / 8;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int hd = A.head_dim;
  float* part = reinterpret_cast<float*>(smem);                 // [4][16][LD]
  float2* ml = reinterpret_cast<float2*>(smem + C::ENDS);       // [4][16]
  float2* mlc = ml + WARPS * 16;                                        // [ROWS] of the CTA
  int* flag = reinterpret_cast<int*>(mlc + C::ROWS);            // [ROWS]
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; e++) {
    float* p = part + (warp * 16 + g + 8 * e) * C::LD + 2 * t4;
#pragma unroll
    for (int n = 0; n < DN; n++) *reinterpret_cast<float2*>(p + n * 8) = make_float2(o[n][2 * e], o[n][2 * e + 1]);
    if (t4 == 0) ml[warp * 16 + g + 8 * e] = make_float2(m[e], l[e]);
  }
  if (tid < C::ROWS) flag[tid] = 0;  // at most 64 rows
  __syncthreads();
  // the key warps of a row into the first of them
  constexpr int Q4 = DP / 4;
  for (int u = tid; u < C::ROWS * Q4; u += C::THREADS) {
    const int r = u / Q4, c = (u % Q4) * 4, w = r / 16, rr = r % 16;
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < KW; k++) top = fmaxf(top, ml[(k * RW + w) * 16 + rr].x);
    const float b = top == -INFINITY ? 0.0f : top;
    float4 sum = make_float4(0, 0, 0, 0);
    float total = 0.0f;
#pragma unroll
    for (int k = 0; k < KW; k++) {
      const float2 x = ml[(k * RW + w) * 16 + rr];
      const float f = ex2((x.x - b) * unit);
      const float4 v = *reinterpret_cast<const float4*>(part + ((k * RW + w) * 16 + rr) * C::LD + c);
      total += x.y * f;
      sum.x += v.x * f;
      sum.y += v.y * f;
      sum.z += v.z * f;
      sum.w += v.w * f;
    }
    *reinterpret_cast<float4*>(part + (w * 16 + rr) * C::LD + c) = sum;
    if (c == 0) mlc[r] = make_float2(top, total);
  }
  if (S > 1) cluster_sync();
  else __syncthreads();
  // the CTAs of the cluster: each finishes every S-th row
  const int mine = (C::ROWS - split + S - 1) / S;
  for (int u = tid; u < mine * Q4; u += C::THREADS) {
    const int r = split + (u / Q4) * S, c = (u % Q4) * 4;
    if (r >= nrows) continue;
    float4 sum;
    float top, total;
    if (S > 1) {
      const uint32_t mla = smem_u32(&mlc[r]), pa = smem_u32(part + r * C::LD + c);
      top = -INFINITY;
      for (int k = 0; k < S; k++) top = fmaxf(top, cluster_load(mla, k));
      const float b = top == -INFINITY ? 0.0f : top;
      sum = make_float4(0, 0, 0, 0);
      total = 0.0f;
      for (int k = 0; k < S; k++) {
        const float f = ex2((cluster_load(mla, k) - b) * unit);
        const float4 v = cluster_load4(pa, k);
        total += cluster_load(mla + 4, k) * f;
        sum.x += v.x * f;
        sum.y += v.y * f;
        sum.z += v.z * f;
        sum.w += v.w * f;
      }
    } else {
      sum = *reinterpret_cast<const float4*>(part + r * C::LD + c);
      top = mlc[r].x;
      total = mlc[r].y;
    }
    const int i = (r0 + r) / A.group, h = hk * A.group + r0 + r - i * A.group;
    const bool none = top == -INFINITY && total == 0.0f;  // a sum that is NaN is kept
    const float inv = none ? 0.0f : 1.0f / total;
    const float4 x = none ? make_float4(0, 0, 0, 0)
                          : make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
    if (c < hd)
      *reinterpret_cast<uint2*>(static_cast<T*>(A.out.data) + (int64_t)(D.q0 + i) * A.out.token +
                                (int64_t)h * A.out.head + c) = make_uint2(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w));
    if (c == 0 && A.lse)
      A.lse[(int64_t)h * A.q_tokens + D.q0 + i] = none ? -INFINITY : log_sum<kMmaLift<T>>(top, unit, total);
    if (!(fabsf(x.x) < INFINITY && fabsf(x.y) < INFINITY && fabsf(x.z) < INFINITY && fabsf(x.w) < INFINITY) &&
        seen(A, D, i) < kend)
      flag[r] = 1;
  }
  __syncthreads();
  for (int r = warp; r < C::ROWS; r += WARPS)
    if (flag[r]) {
      const int i = (r0 + r) / A.group;
      attend_row<T>(A, D, i, hk * A.group + r0 + r - i * A.group, kend, lane);
    }
  if (S > 1) cluster_sync();  // nobody leaves while its shared memory is read
}

// NA: the most axes of a bias, CAP: whether there can be a cap. Where one warp has all keys of a tile
// the registers for both are what limits the CTAs on an SM.
template <typename T, int DP, int RW, int WARPS, int NA, bool CAP>
__global__ void __launch_bounds__(32 * WARPS, MmaCfg<DP, RW, WARPS, NA>::CTAS)
    k_attention_mma(const __grid_constant__ AttnArgs A, const __grid_constant__ CUtensorMap mapK,
                    const __grid_constant__ CUtensorMap mapV) {
  using C = MmaCfg<DP, RW, WARPS>;
  constexpr int KW = C::KW, NT = C::KEYS / 8, DN = DP / 8, DK = DP / 16, PK = C::PV / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* spos = reinterpret_cast<float*>(smem + C::BODY);  // [stage][axis][key]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BARS);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rw = warp % RW, kw = warp / RW, g = lane >> 2, t4 = lane & 3;
  const int S = A.splits;
  const int split = S > 1 ? (int)cluster_rank() : 0;
  const unsigned item = blockIdx.x / S, hgroups = (A.kv_heads + A.cta_heads - 1) / A.cta_heads;
  const int hk0 = (int)(item % hgroups) * A.cta_heads;
  const int hk1 = min(A.kv_heads, hk0 + A.cta_heads);
  const int hd = A.head_dim;
  const float to_cap = A.cap > 0.0f ? A.scale / A.cap : 0.0f;
  const float raw_cap = A.cap / A.scale, unit = A.scale * kLog2e;
  // this lane's place in the 16 x 16 blocks of K and V that ldmatrix takes
  const uint32_t kat = tile_at<DP>(kw * C::KEYS + (lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1);
  const uint32_t vat = tile_at<DP>(kw * C::KEYS + (lane & 7) + (((lane >> 3) & 1) << 3), lane >> 4);
  if (tid == 0) {
    for (int s = 0; s < kMmaStages; s++) mbar_init(&full[s], 1);
    fence_barrier_init();
    tma_prefetch_desc(&mapK);
    tma_prefetch_desc(&mapV);
  }
  pdl_trigger();
  pdl_wait();
  // the stages that are filled and computed next, the phase of the latter; a wait that gave up is
  // not followed by others, but the CTA's barriers are met all the same
  int fstage = 0, stage = 0, flying = 0;  // copies that are not waited for yet (thread 0)
  uint32_t phase = 0;
  bool ok = true;

  int tile;
  Doc D;
  if (!find_document(A, (int)(item / hgroups), C::ROWS, A.group, lane, &D, &tile)) return;
  if ((long long)tile * C::ROWS >= (long long)D.nq * A.group) return;  // the same for all of a cluster
  const int r0 = tile * C::ROWS;  // rows of the document: query * group + head
  const int nrows = D.nq * A.group - r0;
  const int i_first = r0 / A.group;
  const int i_last = min(D.nq - 1, (r0 + C::ROWS - 1) / A.group);
  const int kend = seen(A, D, i_last);   // keys that any row of the tile sees
  const int open = seen(A, D, i_first);  // keys that every row sees
  const int ntiles = (kend + C::TKEYS - 1) / C::TKEYS;
  const int tb = (int)((long long)ntiles * split / S), te = (int)((long long)ntiles * (split + 1) / S);

  // K and V tiles of head after head into the ring; the key positions of a tile, as fp32, through
  // registers and into place a tile later. Where all tiles of a head have a place of their own the
  // positions come once for all heads.
  int ft = tb, fh = hk0;  // the next tile to fetch
  int kraw[2], ref[NA > 0 ? NA : 1];
  const bool stay = te - tb <= kMmaStages;
  auto fetch = [&]() {
    if (fh >= hk1 || tb >= te) return;
    if (tid == 0 && ok) {
      flying++;
      uint8_t* dst = smem + fstage * 2 * C::TILE;
      mbar_arrive_expect_tx(&full[fstage], 2 * C::TILE);
#pragma unroll
      for (int p = 0; p < DP / C::PV; p++) {
        tma_load_3d(dst + p * C::PANEL, &mapK, &full[fstage], p * C::PV, fh, D.k0 + ft * C::TKEYS);
        tma_load_3d(dst + C::TILE + p * C::PANEL, &mapV, &full[fstage], p * C::PV, fh, D.k0 + ft * C::TKEYS);
      }
    }
    if (NA > 0 && A.axes && (!stay || fh == hk0))
#pragma unroll
      for (int x = 0; x < 2; x++) {
        const int u = tid + x * C::THREADS, a = u / C::TKEYS, j = ft * C::TKEYS + u % C::TKEYS;
        if (a < A.axes) kraw[x] = A.kpos[(int64_t)a * A.kv_tokens + D.k0 + min(j, kend - 1)];
      }
  };
  auto fetched = [&]() {  // the positions of the tile last fetched
    if (fh >= hk1 || tb >= te) return;
    if (NA > 0 && A.axes && (!stay || fh == hk0)) {
      float* kp = spos + (stay ? ft - tb : fstage) * (S2S_MAX_AXES * C::TKEYS);
#pragma unroll
      for (int x = 0; x < 2; x++) {
        const int u = tid + x * C::THREADS, a = u / C::TKEYS;
        if (a < A.axes) {
          const int rf = a == 0 ? ref[0] : a == 1 || NA < 3 ? ref[NA > 1] : ref[NA > 2 ? 2 : 0];
          kp[u] = (float)(int)((unsigned)kraw[x] - (unsigned)rf);
        }
      }
    }
    fstage = fstage + 1 == kMmaStages ? 0 : fstage + 1;
    if (++ft == te) {
      ft = tb;
      fh++;
    }
  };
  fetch();

  // this thread's two rows
  int row_seen[2], row_q[2], row_h[2];
  bool live[2];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const int r = r0 + rw * 16 + g + 8 * e;
    live[e] = r - r0 < nrows;
    const int i = live[e] ? r / A.group : i_first;
    row_q[e] = D.q0 + i;
    row_h[e] = live[e] ? r - i * A.group : 0;  // within the key head
    row_seen[e] = live[e] ? seen(A, D, i) : 0;
  }

  // bias: positions count from the tile's first query, so that near ones are exact
  float qpos[2][NA > 0 ? NA : 1];
  if (NA > 0 && A.axes) {
#pragma unroll
    for (int a = 0; a < NA; a++)
      if (a < A.axes) {
        const int* qa = A.qpos + (int64_t)a * A.q_tokens;
        ref[a] = qa[D.q0 + i_first];
#pragma unroll
        for (int e = 0; e < 2; e++) qpos[e][a] = (float)(int)((unsigned)qa[row_q[e]] - (unsigned)ref[a]);
      }
  }

  // Q fragments of a head straight from global memory (rows behind the last read the first)
  uint32_t qf[DK][4], qnext[DK][4];
  const T* qp[2];
  T* op[2];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const int h = hk0 * A.group + row_h[e];
    qp[e] = static_cast<const T*>(A.q.data) + (int64_t)row_q[e] * A.q.token + (int64_t)h * A.q.head + 2 * t4;
    op[e] = static_cast<T*>(A.out.data) + (int64_t)row_q[e] * A.out.token + (int64_t)h * A.out.head + 2 * t4;
  }
  auto load_q = [&]() {
#pragma unroll
    for (int e = 0; e < 2; e++) {
#pragma unroll
      for (int kk = 0; kk < DK; kk++)
#pragma unroll
        for (int x = 0; x < 2; x++)
          qnext[kk][e + 2 * x] =
              kk * 16 + x * 8 < hd ? *reinterpret_cast<const uint32_t*>(qp[e] + kk * 16 + x * 8) : 0u;
      qp[e] += (int64_t)A.group * A.q.head;
    }
  };
  const float per_scale = 1.0f / A.scale;
  float slope[2][NA > 0 ? NA : 1], snext[2][NA > 0 ? NA : 1];
  auto load_slopes = [&](int hk) {
#pragma unroll
    for (int a = 0; a < NA; a++)
      if (a < A.axes)
#pragma unroll
        for (int e = 0; e < 2; e++) snext[e][a] = A.slopes[a * A.q_heads + hk * A.group + row_h[e]];
  };
  load_q();
  load_slopes(hk0);
  fetched();
  fetch();
  __syncthreads();  // the barriers are set up

  bool mend = false;
  for (int hk = hk0; hk < hk1; hk++) {
#pragma unroll
    for (int kk = 0; kk < DK; kk++)
#pragma unroll
      for (int e = 0; e < 4; e++) qf[kk][e] = qnext[kk][e];
#pragma unroll
    for (int a = 0; a < NA; a++)
      if (a < A.axes)
#pragma unroll
        for (int e = 0; e < 2; e++) slope[e][a] = fabsf(snext[e][a]) * per_scale;
    if constexpr (KW == 1)
      if (hk + 1 < hk1) {
        load_q();
        load_slopes(hk + 1);
      }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float o[DN][4];
#pragma unroll
    for (int n = 0; n < DN; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;

    for (int t = tb; t < te; t++) {
      if (ok) {
        ok = attn_wait(A.launch, &full[stage], phase, DEV_TIMEOUT_FULL);
        if (ok) flying--;
        else if (tid == 0)  // nothing is fetched after this
          for (int k = 0; k < flying; k++)
            wait_landed(&full[(stage + k) % kMmaStages], stage + k >= kMmaStages ? phase ^ 1 : phase);
      }
      const int tail = kend - t * C::TKEYS;  // keys of the tile that some row sees
      if (tail < C::TKEYS) {
        // behind them lie other documents' rows, or none: zero weights must not meet what is
        // there, nor may the copies into the stage pass these writes
        for (int u = tid; u < (C::TKEYS - tail) * (DP / 8); u += C::THREADS) {
          const int p = u / ((C::TKEYS - tail) * (C::PV / 8)), c = u % ((C::TKEYS - tail) * (C::PV / 8));
          *reinterpret_cast<uint4*>(smem + stage * 2 * C::TILE + C::TILE + p * C::PANEL +
                                    tail * C::PV * 2 + c * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
      }
      __syncthreads();  // everyone has left the stage that is filled now
      fetched();
      fetch();
      const uint32_t ks = smem_u32(smem + stage * 2 * C::TILE), vs = ks + C::TILE;
      const int j0 = t * C::TKEYS + kw * C::KEYS;
      if (KW == 1 || j0 < kend) {  // some key of this warp is seen
        float s[NT][4];
#pragma unroll
        for (int kk = 0; kk < DK; kk++)
#pragma unroll
          for (int n = 0; n < NT; n += 2) {
            uint32_t b0, b1, b2, b3;
            ldsm_x4(ks + (kk / PK) * C::PANEL + n * 8 * C::PV * 2 + (kat ^ (kk % PK * 32)), b0, b1, b2, b3);
            if (kk == 0) {
              mma_first<T>(s[n], qf[kk], b0, b1);
              mma_first<T>(s[n + 1], qf[kk], b2, b3);
            } else {
              mma_tile<T>(s[n], qf[kk], b0, b1);
              mma_tile<T>(s[n + 1], qf[kk], b2, b3);
            }
          }
        if (CAP && A.cap > 0.0f) capped(reinterpret_cast<float (&)[NT * 4]>(s), to_cap, raw_cap);
        if (NA > 0 && A.axes) {
          const float* kp = spos + (stay ? t - tb : stage) * (S2S_MAX_AXES * C::TKEYS) + kw * C::KEYS + 2 * t4;
#pragma unroll
          for (int a = 0; a < NA; a++)
            if (a < A.axes) {
              const F2 s0 = f2_both(-slope[0][a]), s1 = f2_both(-slope[1][a]);
              const F2 q0 = f2_both(-qpos[0][a]), q1 = f2_both(-qpos[1][a]);
#pragma unroll
              for (int n = 0; n < NT; n++) {
                const F2 k2 = *reinterpret_cast<const F2*>(kp + a * C::TKEYS + n * 8);
                const float2 z0 = f2_unpack(f2_fma(f2_abs(f2_add(k2, q0)), s0, f2_pack(s[n][0], s[n][1])));
                const float2 z1 = f2_unpack(f2_fma(f2_abs(f2_add(k2, q1)), s1, f2_pack(s[n][2], s[n][3])));
                s[n][0] = z0.x;
                s[n][1] = z0.y;
                s[n][2] = z1.x;
                s[n][3] = z1.y;
              }
            }
        }
        if (j0 + C::KEYS > open) {
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (j0 + n * 8 + 2 * t4 + (e & 1) >= row_seen[e >> 1]) s[n][e] = -INFINITY;
        }
        // running maximum (of the scores as they are) and sum
        float keep[2], base[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float top = -INFINITY;
#pragma unroll
          for (int n = 0; n < NT; n++) top = max3(top, s[n][2 * e], s[n][2 * e + 1]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          top = fmaxf(top, m[e]);
          base[e] = top == -INFINITY ? 0.0f : top;  // a row that has seen nothing yet
          keep[e] = ex2((m[e] - base[e]) * unit);
          m[e] = top;
        }
        const F2 u2 = f2_both(unit), lift = f2_both(kMmaLift<T>), b0 = f2_both(-base[0]), b1 = f2_both(-base[1]);
        F2 sum0 = 0, sum1 = 0;  // two zeros each
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const float2 x = f2_unpack(f2_fma(f2_add(f2_pack(s[n][0], s[n][1]), b0), u2, lift));
          const float2 y = f2_unpack(f2_fma(f2_add(f2_pack(s[n][2], s[n][3]), b1), u2, lift));
          s[n][0] = ex2(x.x);
          s[n][1] = ex2(x.y);
          s[n][2] = ex2(y.x);
          s[n][3] = ex2(y.y);
          sum0 = f2_add(sum0, f2_pack(s[n][0], s[n][1]));
          sum1 = f2_add(sum1, f2_pack(s[n][2], s[n][3]));
        }
        const float2 t0 = f2_unpack(sum0), t1 = f2_unpack(sum1);
        l[0] = fmaf(l[0], keep[0], t0.x + t0.y);
        l[1] = fmaf(l[1], keep[1], t1.x + t1.y);
        if (__any_sync(0xffffffffu, keep[0] != 1.0f || keep[1] != 1.0f)) {
#pragma unroll
          for (int n = 0; n < DN; n++) {
            o[n][0] *= keep[0];
            o[n][1] *= keep[0];
            o[n][2] *= keep[1];
            o[n][3] *= keep[1];
          }
        }
        // O += P V; the weights are rounded to the type of v, the sum l is not
#pragma unroll
        for (int kk = 0; kk < NT / 2; kk++) {
          const uint32_t a[4] = {
              pack2<T>(s[2 * kk][0], s[2 * kk][1]), pack2<T>(s[2 * kk][2], s[2 * kk][3]),
              pack2<T>(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack2<T>(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
          for (int n = 0; n < DN; n += 2) {
            uint32_t b0, b1, b2, b3;
            ldsm_x4_t(vs + (n / (2 * PK)) * C::PANEL + kk * 16 * C::PV * 2 + (vat ^ (n % (2 * PK) * 16)), b0, b1,
                      b2, b3);
            mma_tile<T>(o[n], a, b0, b1);
            mma_tile<T>(o[n + 1], a, b2, b3);
          }
        }
      }
      if (++stage == kMmaStages) {
        stage = 0;
        phase ^= 1;
      }
    }
#pragma unroll
    for (int e = 0; e < 2; e++) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
    if (KW == 1 && S == 1)
      mend |= write_rows<T, DN>(A, hk, o, m, l, unit, op, row_q, row_h, live, lane);
    else  // one head (cta_heads is 1)
      join_rows<T, DP, RW, WARPS>(A, D, hk, smem, o, m, l, unit, r0, nrows, kend, S, split);
#pragma unroll
    for (int e = 0; e < 2; e++) op[e] += (int64_t)A.group * A.out.head;
  }
  if (KW == 1 && S == 1 && __any_sync(0xffffffffu, mend)) {
#pragma unroll
    for (int e = 0; e < 2; e++) op[e] -= (int64_t)(hk1 - hk0) * A.group * A.out.head;
    mend_rows<T, DN>(A, D, hk0, hk1, op, row_q, row_h, row_seen, live, kend, lane);
  }
}

template <typename T, int DP, int RW, int WARPS, int NA = S2S_MAX_AXES, bool CAP = true>
cudaError_t launch_attention_mma(AttnArgs& A, cudaStream_t st) {
  using C = MmaCfg<DP, RW, WARPS>;
  auto kernel = k_attention_mma<T, DP, RW, WARPS, NA, CAP>;
  static LaunchSetup setup;
  int ctas = 0;
  cudaError_t err = resident_ctas(setup, kernel, C::THREADS, C::SMEM, &ctas);
  if (err != cudaSuccess) return err;
  set_slots(A, C::ROWS, A.group);
  const long long tiles = (long long)A.slots * A.kv_heads;
  // The keys of a tile are split over a cluster until there are twice the CTAs that fit on the
  // device, which evens out documents of different lengths, with eight tiles of keys or more
  // for each (by the mean length: the host does not know the offsets); or with one, while that
  // is all that half fills the device.
  const long long ktiles = (A.kv_tokens / A.documents + C::TKEYS - 1) / C::TKEYS;
  int splits = 1;
  while (splits < kMaxSplits && (tiles * splits < ctas / 2 ? ktiles >= 2 * splits
                                                           : tiles * splits < 2LL * ctas && ktiles >= 16 * splits))
    splits *= 2;
  A.splits = splits;
  // many tiles: a CTA takes several heads of a tile, the next head's loads under way while it
  // computes, as long as three rounds of CTAs are left
  A.cta_heads = 1;
  if (C::KW == 1 && splits == 1)
    A.cta_heads = (int)std::max(1LL, std::min((long long)A.kv_heads, tiles / (3LL * ctas)));
  const long long items = (long long)A.slots * ((A.kv_heads + A.cta_heads - 1) / A.cta_heads);
  const long long grid = items * splits;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof cfg);
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (splits > 8) {  // beyond the portable size
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (err != cudaSuccess) return err;
  }
  if (splits > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = splits;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap k, v;
  memset(&k, 0, sizeof k);
  memset(&v, 0, sizeof v);
  if (A.kv_tokens > 0 &&
      (!make_map_heads(&k, A.k, BF16, A.kv_tokens, A.kv_heads, A.head_dim, C::TKEYS, C::PV) ||
       !make_map_heads(&v, A.v, BF16, A.kv_tokens, A.kv_heads, A.head_dim, C::TKEYS, C::PV)))
    return cudaErrorInvalidValue;
  return cudaLaunchKernelEx(&cfg, kernel, A, k, v);
}

template <typename T, int DP>
cudaError_t launch_attention_mma(AttnArgs& A, cudaStream_t st) {
  // The fewest row warps that hold the mean document's rows; fewer still where the tiles, split
  // as far as they go, would not fill the device (K and V are then read again, from L2). Where
  // even so there is at most one CTA for an SM, it has eight warps and tiles of 128 keys.
  const long long rows = (long long)A.q_tokens * A.group, mean = rows / A.documents;
  auto ctas = [&](int n) { return (rows / n + A.documents) * A.kv_heads * kMaxSplits; };
  const bool wide = ctas(16) <= 148 && A.kv_tokens / A.documents >= 1024;
  if (mean <= 16 || ctas(32) < 148)
    return wide ? launch_attention_mma<T, DP, 1, 8>(A, st) : launch_attention_mma<T, DP, 1, 4>(A, st);
  if (mean <= 32 || ctas(64) < 148) return launch_attention_mma<T, DP, 2, 4>(A, st);
  if (A.cap > 0.0f)
    return A.axes == 0   ? launch_attention_mma<T, DP, 4, 4, 0, true>(A, st)
           : A.axes <= 2 ? launch_attention_mma<T, DP, 4, 4, 2, true>(A, st)
                         : launch_attention_mma<T, DP, 4, 4, 3, true>(A, st);
  return A.axes == 0   ? launch_attention_mma<T, DP, 4, 4, 0, false>(A, st)
         : A.axes <= 2 ? launch_attention_mma<T, DP, 4, 4, 2, false>(A, st)
                       : launch_attention_mma<T, DP, 4, 4, 3, false>(A, st);
}

template <typename T>
cudaError_t launch_attention_mma(AttnArgs& A, cudaStream_t st) {
  return A.head_dim <= 32   ? launch_attention_mma<T, 32>(A, st)
         : A.head_dim <= 64 ? launch_attention_mma<T, 64>(A, st)
                            : launch_attention_mma<T, 128>(A, st);
}

}  // namespace
}  // namespace s2s
