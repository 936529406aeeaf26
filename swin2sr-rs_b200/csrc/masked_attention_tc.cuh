// The attention of masked_attention.cu on tcgen05, for documents with many queries.
//
// A CTA takes 256 query rows of one document and head as two tiles of 128, which share every
// K and V tile that TMA brings in. Two groups of four warps do the softmax of the two tiles; of
// a third group one warp loads and one issues the MMAs:
//   S = Q_w K_i^T        both operands from shared memory, S in one of the score buffers in TMEM
//   softmax group w      reads S, a row per thread, and writes the weights P as 16-bit values
//                        over the first half of S's columns
//   O_w += P V_i         P from TMEM, V_i as it lies in memory (keys by values: the MN-major
//                        operand form), O_w in TMEM
// The score products run ahead of the softmax: three buffers of 128 keys for head_dim <= 64, four
// of 64 keys beyond (TMEM holds 512 columns, of which the outputs take 128 or 256). With one
// buffer a tile, each group's softmax (1900 cycles) waited for its own two products and they for
// it, 3200-3400 cycles a round.
//
// The output is scaled again only when a row's maximum grows by more than 2^8 beyond the one its
// weights refer to (weights then stay below 2^8, in the range of both types, and the sums are
// 32-bit), which after the first tiles is rare; the group does it itself.
#pragma once

namespace s2s {
namespace {

constexpr int kTcTile = 128;     // rows of a tile
constexpr int kTcThreads = 384;

template <int NP>  // panels of 64 values: head_dim <= 64 * NP
struct TcCfg {
  static constexpr int BN = NP == 1 ? 128 : 64;      // keys of a tile
  static constexpr int NB = NP == 1 ? 3 : 4;         // score buffers
  static constexpr int OUT = NB * BN;                // TMEM column of the outputs
  static constexpr int QB = NP * kTcTile * 128;      // bytes of a Q tile
  static constexpr int KB = NP * BN * 128;           // of a K or V tile
  static constexpr int STAGES = 4;                   // of K, and of V
  static constexpr int KRING = 2 * QB;
  static constexpr int VRING = KRING + STAGES * KB;
  static constexpr int POS = VRING + STAGES * KB;
  static constexpr int BARS = POS + 2 * 2 * S2S_MAX_AXES * BN * 4;
  static constexpr int NBARS = 4 * STAGES + 3 * NB + 4;
  static constexpr int SMEM = BARS + NBARS * 8 + 16 + 1024;  // + alignment
};

// Instruction descriptor: fp16 or bf16 operands, fp32 sums; B K-major, or MN-major.
__device__ __forceinline__ uint32_t idesc_16(int M, int N, bool bf16, bool b_mn) {
  return idesc_f16_f32(M, N) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u);
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Values of a TMEM load are not used before this point (after the wait for the load).
__device__ __forceinline__ void loaded(uint32_t (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]),
                      "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}

// What an MMA costs the issuing warp counts: it shares a scheduler with two softmax warps. All lanes
// run the loop, steered by values that the compiler knows to be uniform, and an elected one issues;
// descriptors are the 32-bit word that varies and a constant, predicates are constants but for the
// first of an output product. An MMA then takes 22 cycles to issue; in a loop of one lane, or with
// whole descriptors, 85 to 130, more than its execution.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one;
}
// High words: groups of eight rows 1024 bytes apart, descriptor version, 128-byte swizzle.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lead) {
  return ((saddr >> 4) & 0x3FFFu) | (lead >> 4) << 16;
}
template <bool ACC>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "n"(ACC ? 1 : 0), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, 1, 0;\n\t"
      "mov.b64 b, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "n"(kDescHigh)
      : "memory");
}

// 2^x of two values on the multiply-add pipe: x = n + f with n the nearest whole number (by
// adding 1.5 2^23, after which n is in the low bits), 2^f by the polynomial of degree 4 of least
// relative error on [-1/2, 1/2] (2.6e-6; the weights are rounded to 2^-9 or 2^-12 next), n into
// the exponent. Below 2^-125 it stays there.
__device__ __forceinline__ F2 ex2_poly(F2 x) {
  const float2 xs = f2_unpack(x);
  const F2 c = f2_pack(fmaxf(xs.x, -125.0f), fmaxf(xs.y, -125.0f));
  const F2 t = f2_add(c, f2_both(12582912.0f));
  const F2 f = f2_add(c, f2_fma(t, f2_both(-1.0f), f2_both(12582912.0f)));
  F2 p = f2_fma(f2_both(0.009570102207362652f), f, f2_both(0.05591785907745361f));
  p = f2_fma(p, f, f2_both(0.240247443318367f));
  p = f2_fma(p, f, f2_both(0.6931217908859253f));
  p = f2_fma(p, f, f2_both(0.9999992847442627f));
  const float2 n = f2_unpack(t), y = f2_unpack(p);
  return f2_pack(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(n.x) << 23)),
                 __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(n.y) << 23)));
}

template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ void group_sync(int id) {
  asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory");
}

// The products of a CTA in the order they are issued: tile 0 and 1 in turn, for key tile after
// key tile, the one with more of them alone at the end.
struct TcStep {
  int w, i;
  __device__ __forceinline__ TcStep(int n0) : w(n0 > 0 ? 0 : 1), i(0) {}
  __device__ __forceinline__ void next(int n0, int n1) {
    if (w == 0 && i < n1) {
      w = 1;
    } else {
      i++;
      w = i < n0 ? 0 : 1;
    }
  }
};

// PLAIN: no cap, no bias.
template <typename T, int NP, bool PLAIN>
__global__ void __launch_bounds__(kTcThreads, 1)
    k_attention_tc(const __grid_constant__ AttnArgs A, const __grid_constant__ CUtensorMap mapQ,
                   const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV) {
  using C = TcCfg<NP>;
  constexpr int BN = C::BN, NB = C::NB, ST = C::STAGES;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sQ = smem;
  uint8_t* kring = smem + C::KRING;
  uint8_t* vring = smem + C::VRING;
  float* spos = reinterpret_cast<float*>(smem + C::POS);  // [group][buffer][axis][key]
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + C::BARS);  // [stage]
  uint64_t* k_empty = k_full + ST;
  uint64_t* v_full = k_empty + ST;
  uint64_t* v_empty = v_full + ST;
  uint64_t* s_full = v_empty + ST;  // [score buffer]
  uint64_t* p_full = s_full + NB;
  uint64_t* o_done = p_full + NB;   // the output product that read the buffer's weights is complete
  uint64_t* q_full = o_done + NB;   // [tile]
  uint64_t* fin = q_full + 2;       // [scores, outputs]: every product has retired
  uint32_t* holder = reinterpret_cast<uint32_t*>(fin + 2);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int s = 0; s < ST; s++) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int b = 0; b < NB; b++) {
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], 4);
      mbar_init(&o_done[b], 1);
    }
    for (int w = 0; w < 2; w++) mbar_init(&q_full[w], 1);
    mbar_init(&fin[0], 1);
    mbar_init(&fin[1], 1);
    fence_barrier_init();
    tma_prefetch_desc(&mapQ);
    tma_prefetch_desc(&mapK);
    tma_prefetch_desc(&mapV);
  }
  if (warp == 9) {
    tmem_alloc(holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *holder;
  pdl_trigger();
  pdl_wait();

  // The slots from the back: in causal order the last tiles have the most keys.
  const int slot = A.slots - 1 - (int)(blockIdx.x / A.q_heads), h = blockIdx.x % A.q_heads;
  const int hk = h / A.group;
  int tile = 0;
  Doc D;
  // the CTA's first query; slots behind the document's last tile have none
  const bool any = find_document(A, slot, 2 * kTcTile, 1, lane, &D, &tile) &&
                   (long long)tile * (2 * kTcTile) < D.nq;
  const int i0 = any ? tile * (2 * kTcTile) : D.nq;
  int rows[2], kend[2], n[2];
#pragma unroll
  for (int w = 0; w < 2; w++) {
    rows[w] = max(0, min(kTcTile, D.nq - i0 - w * kTcTile));
    kend[w] = rows[w] > 0 ? seen(A, D, i0 + w * kTcTile + rows[w] - 1) : 0;
    n[w] = (kend[w] + BN - 1) / BN;
  }
  const int kmax = max(kend[0], kend[1]);
  const int ksteps = (A.head_dim + 15) / 16;

  // registers: 384 threads begin with 168 each; the softmax groups take what the third gives
  // (2 * 128 * 200 + 128 * 96 = 63488 of 64512)
  if (warp >= 8) {
    fewer_registers<96>();
    if (warp == 8 && lane == 0) {
      // ------------------------------------------------------------------ loads
      auto load = [&](uint8_t* dst, int bytes, const CUtensorMap* map, uint64_t* bar, int head, int row) {
        mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
        for (int p = 0; p < NP; p++) tma_load_3d(dst + p * (bytes / NP), map, bar, p * 64, head, row);
      };
      const int N = max(n[0], n[1]);
      bool ok = true;
      int i = 0;
      for (; i < N && ok; i++) {
        const int s = i % ST;
        if (i >= ST) ok = mbar_wait(&k_empty[s], ((i / ST) - 1) & 1, DEV_TIMEOUT_EMPTY);
        if (!ok) break;
        load(kring + s * C::KB, C::KB, &mapK, &k_full[s], hk, D.k0 + i * BN);
        if (i == 0)
          for (int w = 0; w < 2; w++)
            if (n[w] > 0) load(sQ + w * C::QB, C::QB, &mapQ, &q_full[w], h, D.q0 + i0 + w * kTcTile);
        if (i >= ST) ok = mbar_wait(&v_empty[s], ((i / ST) - 1) & 1, DEV_TIMEOUT_EMPTY);
        if (ok) load(vring + s * C::KB, C::KB, &mapV, &v_full[s], hk, D.k0 + i * BN);
      }
      // no copy is in flight when the CTA ends, also where a wait gave up
      if (N > 0)
        for (int w = 0; w < 2; w++)
          if (n[w] > 0) mbar_wait(&q_full[w], 0, DEV_TIMEOUT_FULL);
      for (int k = max(0, i - ST); k < i; k++) {
        mbar_wait(&k_full[k % ST], (k / ST) & 1, DEV_TIMEOUT_FULL);
        if (ok || k < i - 1) mbar_wait(&v_full[k % ST], (k / ST) & 1, DEV_TIMEOUT_FULL);
      }
    }
    // values that steer the products, from reductions, which give uniform registers
    const int n0 = (int)__reduce_max_sync(0xffffffffu, (unsigned)n[0]);
    const int n1 = (int)__reduce_max_sync(0xffffffffu, (unsigned)n[1]);
    const int keys = (int)__reduce_max_sync(0xffffffffu, (unsigned)kmax);
    const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
    const int total = n0 + n1, last = max(n0, n1) - 1;
    bool ok = true;
    auto wait = [&](uint64_t* bar, int phase, unsigned code) {
      ok = __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, code));
    };
    if (warp == 9) {
      // ----------------------------------------------------------- score products
      const uint32_t one = elect_one(), id = idesc_16(128, BN, BF16, false);
      const uint32_t dq = desc_low(smem_u32(sQ), 16), dk = desc_low(smem_u32(kring), 16);
      TcStep s(n0);
      for (int p = 0, b = 0, ph = 1; p < total; p++, s.next(n0, n1)) {
        const int st = s.i % ST;
        if (p >= NB) wait(&o_done[b], ph, DEV_TIMEOUT_ACC);
        if (ok && (s.w == 0 || s.i >= n0)) wait(&k_full[st], s.i / ST, DEV_TIMEOUT_FULL);
        if (ok && s.i == 0) wait(&q_full[s.w], 0, DEV_TIMEOUT_FULL);
        if (!ok) break;
        tc_fence_after();
        const uint32_t q = dq + s.w * (C::QB >> 4), k = dk + st * (C::KB >> 4), d = tm + b * BN;
        if (one) {
          mma_ss<false>(d, q, k, id);
#pragma unroll
          for (int c = 1; c < 4 * NP; c++)
            if (c < ksteps)
              mma_ss<true>(d, q + (((c >> 2) * kTcTile * 128 + (c & 3) * 32) >> 4),
                           k + (((c >> 2) * BN * 128 + (c & 3) * 32) >> 4), id);
          tc_commit(&s_full[b]);
          if (s.w == 1 || s.i >= n1) tc_commit(&k_empty[st]);  // the K tile's last use
        }
        __syncwarp();
        if (++b == NB) {
          b = 0;
          ph ^= 1;
        }
      }
      if (one) tc_commit(&fin[0]);
      __syncwarp();
      mbar_wait(&fin[0], 0, DEV_TIMEOUT_ACC);
    } else if (warp == 10) {
      // ---------------------------------------------------------- output products
      // V is read along its rows as the contraction (keys contract, values are the N extent):
      // panels of 64 values BN * 128 bytes apart
      const uint32_t one = elect_one(), id = idesc_16(128, ksteps * 16, BF16, true);
      const uint32_t dv = desc_low(smem_u32(vring), BN * 128);
      TcStep s(n0);
      for (int p = 0, b = 0, ph = 0; p < total; p++, s.next(n0, n1)) {
        const int st = s.i % ST, tail = keys - last * BN, steps = (tail + 15) / 16;
        if (s.w == 0 || s.i >= n0) {
          wait(&v_full[st], s.i / ST, DEV_TIMEOUT_FULL);
          if (s.i == last && tail % 16) {
            // Keys that no row sees, and rows of other documents behind them, have zero weights:
            // what lies there must not reach the product, which takes keys by 16.
            for (int x = 0; x < NP; x++)
              for (int c = tail * 8 + lane; c < steps * 16 * 8; c += 32)
                *reinterpret_cast<uint4*>(vring + st * C::KB + x * BN * 128 + c * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
        if (ok) wait(&p_full[b], ph, DEV_TIMEOUT_ACC);
        if (!ok) break;
        tc_fence_after();
        const uint32_t v = dv + st * (C::KB >> 4), d = tm + C::OUT + s.w * 64 * NP, w = tm + b * BN;
        if (one) {
          mma_ts(d, w, v, id, s.i != 0);
          if (s.i < last) {
#pragma unroll
            for (int c = 1; c < BN / 16; c++) mma_ts(d, w + c * 8, v + c * (2048 >> 4), id);
          } else {
            for (int c = 1; c < steps; c++) mma_ts(d, w + c * 8, v + c * (2048 >> 4), id);
          }
          tc_commit(&o_done[b]);
          if (s.w == 1 || s.i >= n1) tc_commit(&v_empty[st]);  // the V tile's last use
        }
        __syncwarp();
        if (++b == NB) {
          b = 0;
          ph ^= 1;
        }
      }
      if (one) tc_commit(&fin[1]);
      __syncwarp();
      mbar_wait(&fin[1], 0, DEV_TIMEOUT_ACC);
    }
  } else {
    more_registers<200>();
    // ------------------------------------------------------------------ softmax
    const int w = warp >> 2, r = tid & 127;
    const int rows_w = w ? rows[1] : rows[0], n_w = w ? n[1] : n[0];
    const int i = i0 + w * kTcTile + r;       // this thread's query
    const bool live = r < rows_w;
    const int mine = live ? seen(A, D, i) : 0;
    const int open = rows_w > 0 ? seen(A, D, i0 + w * kTcTile) : 0;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t to = lanes + C::OUT + w * 64 * NP;
    const float unit = A.scale * kLog2e, raw_cap = A.cap / A.scale;
    const float to_cap = A.cap > 0.0f ? A.scale / A.cap : 0.0f;
    bool ok = true;
    float m = -INFINITY, l = 0.0f;

    // bias: slope times position for this row's query (from the CTA's first query on) and,
    // in shared memory, for the keys of a tile, each loaded a tile ahead by one thread
    float qf[S2S_MAX_AXES], slope[S2S_MAX_AXES];
    int ref[S2S_MAX_AXES], kraw[S2S_MAX_AXES];
    float* pos = spos + w * 2 * S2S_MAX_AXES * BN;
    auto key_positions = [&](int t) {
      const int j = t * BN + r;
      if (r < BN)
#pragma unroll
        for (int a = 0; a < S2S_MAX_AXES; a++)
          if (a < A.axes) kraw[a] = j < D.nk ? A.kpos[(int64_t)a * A.kv_tokens + D.k0 + j] : ref[a];
    };
    if (!PLAIN && n_w > 0) {
#pragma unroll
      for (int a = 0; a < S2S_MAX_AXES; a++)
        if (a < A.axes) {
          const int* qa = A.qpos + (int64_t)a * A.q_tokens + D.q0;
          ref[a] = qa[i0];
          slope[a] = fabsf(A.slopes[a * A.q_heads + h]) / A.scale;
          qf[a] = slope[a] * (float)(int)((unsigned)qa[live ? i : i0] - (unsigned)ref[a]);
        }
      key_positions(0);
    }

    // The place of this group's tile t in the order of the products (TcStep): its buffer and phase.
    // A group waits for its last output product only where it needs the outputs. That cannot be
    // one phase off: a score product waited for the output product NB places before it, output
    // products are in order, and behind this group's tile t there are fewer than NB of the other's
    // before the group's next (at the end too: tile 1 has at most 128 / BN key tiles more).
    auto place = [&](int t) { return min(t, n[0]) + min(t, n[1]) + (w & (t < n[0] ? 1 : 0)); };
    auto output_done = [&](int t) {
      const int q = place(t);
      if (ok) ok = mbar_wait(&o_done[q % NB], (q / NB) & 1, DEV_TIMEOUT_ACC);
      __syncwarp();
      tc_fence_after();
    };

    for (int t = 0; t < n_w; t++) {
      const int q = place(t), b = q % NB;
      const uint32_t ts = lanes + b * BN;
      const float* kp = pos + (t & 1) * S2S_MAX_AXES * BN;
      if (!PLAIN && A.axes) {
        if (r < BN)
#pragma unroll
          for (int a = 0; a < S2S_MAX_AXES; a++)
            if (a < A.axes)
              const_cast<float*>(kp)[a * BN + r] = slope[a] * (float)(int)((unsigned)kraw[a] - (unsigned)ref[a]);
        group_sync(1 + w);
        if (t + 1 < n_w) key_positions(t + 1);
      }
      // after a wait that gave up the group goes on without waiting, so that its four warps
      // still meet at their barrier
      if (ok) ok = mbar_wait(&s_full[b], (q / NB) & 1, DEV_TIMEOUT_ACC);
      tc_fence_after();
      uint32_t s[BN / 32][32];
#pragma unroll
      for (int c = 0; c < BN / 32; c++) tmem_ld32_nw(ts + c * 32, s[c]);
      tc_wait_ld();
#pragma unroll
      for (int c = 0; c < BN / 32; c++) loaded(s[c]);
      auto at = [&](int j) -> float { return __uint_as_float(s[j >> 5][j & 31]); };
      auto set = [&](int j, float x) { s[j >> 5][j & 31] = __float_as_uint(x); };

      if (!PLAIN) {
        if (A.cap > 0.0f) {
#pragma unroll
          for (int c = 0; c < BN / 32; c++) capped(reinterpret_cast<float (&)[32]>(s[c]), to_cap, raw_cap);
        }
#pragma unroll
        for (int a = 0; a < S2S_MAX_AXES; a++)
          if (a < A.axes) {
            const F2 q2 = f2_both(-qf[a]);
#pragma unroll
            for (int j = 0; j < BN; j += 4) {
              const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(kp + a * BN + j);
              const float2 x = f2_unpack(f2_add(k.x, q2)), y = f2_unpack(f2_add(k.y, q2));
              set(j, at(j) - fabsf(x.x));
              set(j + 1, at(j + 1) - fabsf(x.y));
              set(j + 2, at(j + 2) - fabsf(y.x));
              set(j + 3, at(j + 3) - fabsf(y.y));
            }
          }
      }
      if ((t + 1) * BN > open) {
        const int last = mine - t * BN;
#pragma unroll
        for (int j = 0; j < BN; j++)
          if (j >= last) set(j, -INFINITY);
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < BN; j += 2) top[(j >> 1) & 3] = max3(top[(j >> 1) & 3], at(j), at(j + 1));
      const float high = fmaxf(max3(top[0], top[1], top[2]), top[3]) * unit;
      if (t == 0) {
        m = high;
      } else if (__any_sync(0xffffffffu, high > m + 8.0f)) {
        const float next = fmaxf(m, high), keep = next == -INFINITY ? 1.0f : ex2(m - next);
        m = next;
        l *= keep;
        // the output product before this tile's is complete, this one waits for the weights
        output_done(t - 1);
        for (int c = 0; c < ksteps * 16; c += 16) {
          uint32_t o[16];
          tmem_ld16(to + c, o);
#pragma unroll
          for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
          tmem_st16(to + c, o);
        }
      }
      const F2 base2 = f2_both(m == -INFINITY ? 0.0f : -m), unit2 = f2_both(unit);
      F2 sum[2] = {0, 0};  // two zeros each
#pragma unroll
      for (int c = 0; c < BN / 64; c++) {
        uint32_t p[32];
#pragma unroll
        for (int j = 0; j < 32; j++) {
          F2 x = f2_fma(f2_pack(at(64 * c + 2 * j), at(64 * c + 2 * j + 1)), unit2, base2);
          if (j % 4 == 3) {
            x = ex2_poly(x);
          } else {
            const float2 xs = f2_unpack(x);
            x = f2_pack(ex2(xs.x), ex2(xs.y));
          }
          sum[j & 1] = f2_add(sum[j & 1], x);
          const float2 y = f2_unpack(x);
          p[j] = pack2<T>(y.x, y.y);
        }
        tmem_st32(ts + c * 32, p);
      }
      const float2 total = f2_unpack(f2_add(sum[0], sum[1]));
      l += total.x + total.y;
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[b]);
    }

    // ------------------------------------------------------------------- output
    if (n_w > 0) output_done(n_w - 1);
    const bool none = m == -INFINITY;
    const float inv = none ? 0.0f : 1.0f / l;
    float check = 0.0f;  // NaN where an output is NaN or infinite
    T* out = static_cast<T*>(A.out.data) + (int64_t)(D.q0 + i) * A.out.token + (int64_t)h * A.out.head;
    if (rows_w > 0)
      for (int c = 0; c < ksteps * 16; c += 16) {
        uint32_t o[16];
        if (n_w > 0) tmem_ld16(to + c, o);
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float x = n_w > 0 ? __uint_as_float(o[2 * e]) * inv : 0.0f;
          const float y = n_w > 0 ? __uint_as_float(o[2 * e + 1]) * inv : 0.0f;
          check = fmaf(x, 0.0f, fmaf(y, 0.0f, check));
          v[e] = pack2<T>(x, y);
        }
        if (live) {
          *reinterpret_cast<uint4*>(out + c) = make_uint4(v[0], v[1], v[2], v[3]);
          if (c + 8 < A.head_dim) *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(v[4], v[5], v[6], v[7]);
        }
      }
    if (live && A.lse)
      A.lse[(int64_t)h * A.q_tokens + D.q0 + i] = none ? -INFINITY : (m + log2f(l)) * kLn2;
    // keys of the document that this row does not see had zero weights: a NaN or infinity
    // among their values shows here, and the row is done again without them
    unsigned redo = __ballot_sync(0xffffffffu, check != 0.0f && live && mine < kmax);
    __syncwarp();
    while (redo) {
      const int src = __ffs(redo) - 1;
      redo &= redo - 1;
      attend_row<T>(A, D, i0 + w * kTcTile + (warp & 3) * 32 + src, h, lane);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

template <typename T, int NP, bool PLAIN>
cudaError_t launch_attention_tc(AttnArgs& A, cudaStream_t st) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  using C = TcCfg<NP>;
  auto kernel = k_attention_tc<T, NP, PLAIN>;
  static LaunchSetup setup;
  int ctas = 0;
  const cudaError_t err = resident_ctas(setup, kernel, kTcThreads, C::SMEM, &ctas);
  if (err != cudaSuccess) return err;
  CUtensorMap q, k, v;
  if (!make_map_heads(&q, A.q, BF16, A.q_tokens, A.q_heads, A.head_dim, kTcTile, 64) ||
      !make_map_heads(&k, A.k, BF16, A.kv_tokens, A.kv_heads, A.head_dim, C::BN, 64) ||
      !make_map_heads(&v, A.v, BF16, A.kv_tokens, A.kv_heads, A.head_dim, C::BN, 64))
    return cudaErrorInvalidValue;
  set_slots(A, 2 * kTcTile, 1);
  const long long grid = (long long)A.slots * A.q_heads;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  return launch_pdl(kernel, dim3((unsigned)grid), dim3(kTcThreads), C::SMEM, st, A, q, k, v);
}

template <typename T>
cudaError_t launch_attention_tc(AttnArgs& A, cudaStream_t st) {
  const bool plain = A.cap == 0.0f && A.axes == 0;
  if (A.head_dim <= 64)
    return plain ? launch_attention_tc<T, 1, true>(A, st) : launch_attention_tc<T, 1, false>(A, st);
  return plain ? launch_attention_tc<T, 2, true>(A, st) : launch_attention_tc<T, 2, false>(A, st);
}

}  // namespace
}  // namespace s2s
