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
// The score products run ahead of the softmax. TMEM holds 512 columns, of which the outputs take 128
// or 256: for head_dim <= 64 three score buffers of 128 keys serve both tiles in turn, beyond it
// each tile has two of 64 keys. With one buffer of 128 keys a tile, each group's softmax (1900
// cycles) waited for its own two products and they for it, 3200-3400 cycles a round.
//
// The output is scaled again only when a row's maximum grows by more than 2^8 beyond the one its
// weights refer to, which after the first tiles is rare; the group does it itself. Weights then stay
// below 2^8, in fp16 with its lift (kTcLift) below 2^15, and the sums are 32-bit.
//
// Bound: without a cap or a bias, for head_dim <= 64 the special function unit (16 exponentials a cycle
// and SM: 2048 cycles for 256 x 128 pairs, of 2900), beyond it the tensor core with its 64-key score
// products. With either no unit is full (six images with two axes: exponentials 0.40, issue 0.48, tensor
// 0.20 of the cycles): two softmax warps a scheduler, each a chain from scores to weights. Measured
// (B200, bf16, non-causal, 37 heads, 4096 x 4096, replayed from a graph): 194 us at head 64, 820 TFLOP/s;
// 288 us at head 128, 1100 TFLOP/s, 0.67 of the measured bf16 burst; with a cap of 50 340 and 406 us, with
// one, two, three axes of bias 334, 333, 463 and 417, 424, 504. Causal 16384, eight heads of 128: 446-457
// us in bursts, 1220 TFLOP/s, 530 back to back for seconds under the power cap, 1040 TFLOP/s.
#pragma once

namespace s2s {
namespace {

constexpr int kTcTile = 128;     // rows of a tile
constexpr int kTcThreads = 384;

template <int NP>  // panels of 64 values: head_dim <= 64 * NP
struct TcCfg {
  static constexpr int BN = NP == 1 ? 128 : 64;      // keys of a tile
  static constexpr int NB = NP == 1 ? 3 : 4;         // score buffers
  static constexpr int SW = NP;                      // warps that issue score products
  static constexpr int OUT = NB * BN;                // TMEM column of the outputs
  static constexpr int QB = NP * kTcTile * 128;      // bytes of a Q tile
  static constexpr int KB = NP * BN * 128;           // of a K or V tile
  static constexpr int STAGES = 4;                   // of K, and of V
  static constexpr int KRING = 2 * QB;
  static constexpr int VRING = KRING + STAGES * KB;
  static constexpr int POS = VRING + STAGES * KB;
  static constexpr int BARS = POS + 2 * 2 * S2S_MAX_AXES * BN * 4;
  static constexpr int NBARS = 4 * STAGES + 3 * NB + 13;
  static constexpr int SMEM = BARS + NBARS * 8 + 16 + 1024;  // + alignment
};

// Instruction descriptor: fp16 or bf16 operands, fp32 sums; B K-major, or MN-major.
__device__ __forceinline__ uint32_t idesc_16(int M, int N, bool bf16, bool b_mn) {
  return idesc_f16_f32(M, N) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u);
}

// 32 lanes x 32 columns from registers into TMEM; tc_wait_st waits for the store.
__device__ __forceinline__ void tmem_st32_nw(uint32_t taddr, const uint32_t (&r)[32]) {
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
// The fragments of mma.sync in TMEM: 16 lanes x 64 fp32 columns, thread 4 g + t holding of each 8
// columns 2 t and 2 t + 1 of rows g and g + 8; and 16 lanes x 32 columns of 16-bit pairs, pair t of
// each 4 columns of rows g and g + 8.
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_frag(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
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
// Weights are 2^(s unit - m unit), in one multiply-add behind the rounded m unit, which all weights of a
// row share. Beyond this size (in either direction), where that rounding passes the 2^-12 that a score has
// itself, m is taken off first. (Taken off first in all rows: six images 307 -> 325 us, causal 16384 511 ->
// 539 back to back.)
constexpr float kLargeScore = 4096.0f;
// In fp16 weights are 2^7 times as large, so that those down to 2^-31 of the largest count in the second
// product (its least value is 2^-24; see kMmaLift).
template <typename T>
constexpr float kTcLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;
// What a row's exponents lose when its maximum grows from m to `next`.
__device__ __forceinline__ float growth(float m, float next, float unit) {
  const float a = m * unit, b = next * unit;
  return fmaxf(fabsf(a), fabsf(b)) < kLargeScore ? a - b : (m - next) * unit;
}

// Where the products of key tile i and row tile w have their place: score buffer and the parity of
// its use. Three buffers are taken in the order of the products, tile 0 and 1 in turn and at the
// end the one that has more (n0, n1: their key tiles); of four each tile has two.
//
// Every wait is at most one phase from the one waited for. A score product into a buffer waits for
// the output product that read it last. Output products are in order, also across the tiles; none
// starts before its group's weights, which are made from these scores. So between two uses of a
// buffer whoever waits for the first is through. At the end of tile 0, tile 1 has at most 128 / BN
// key tiles more, fewer than buffers, so that an output product waited for there is not passed.
template <int NB>
struct TcPlace {
  int buffer, parity;
  __device__ __forceinline__ TcPlace(int w, int i, int n0, int n1) {
    if (NB == 4) {
      buffer = 2 * w + (i & 1);
      parity = (i >> 1) & 1;
    } else {
      const int q = min(i, n0) + min(i, n1) + (i < n0 ? w : 0);
      buffer = q % NB;
      parity = (q / NB) & 1;
    }
  }
};

// The loader's schedule: key and value tiles in turn through rings of STAGES each, `released` a wait for
// the stage of an earlier tile, which may give up. At the end every copy that its stage's next tile did
// not wait for is waited for, also then: none is in flight when the CTA ends.
#pragma nv_exec_check_disable
template <int STAGES, typename Released, typename Copy, typename Landed>
__host__ __device__ __forceinline__ void load_tiles(int tiles, Released&& released, Copy&& copy, Landed&& landed) {
  int n[2] = {0, 0};  // copies of keys, of values
  for (int i = 0; i < 2 * tiles; i++) {
    const bool value = i & 1;
    if (i / 2 >= STAGES && !released(value, i / 2)) break;
    copy(value, i / 2);
    n[i & 1]++;
  }
  for (int v = 0; v < 2; v++)
    for (int i = n[v] > STAGES ? n[v] - STAGES : 0; i < n[v]; i++) landed(v == 1, i);
}

// MODE 0: no cap, no bias; 1 + axes: a bias of one to three axes, with or without a cap; 1: a cap that keeps
// scores below kLargeScore, 5: any cap. (With what large scores take, 37 heads of 64 x 4096^2 under a cap of
// 50 are 353 us instead of 331.)
template <typename T, int NP, int MODE>
__global__ void __launch_bounds__(kTcThreads, 1)
    k_attention_tc(const __grid_constant__ AttnArgs A, const __grid_constant__ CUtensorMap mapQ,
                   const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV) {
  using C = TcCfg<NP>;
  constexpr int BN = C::BN, NB = C::NB, ST = C::STAGES;
  constexpr bool BIAS = MODE >= 2 && MODE <= 4, CAP = MODE == 1 || MODE == 5;
  constexpr int NA = BIAS ? MODE - 1 : 1;  // axes of a bias
  using Place = TcPlace<NB>;
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
  uint64_t* fin = q_full + 2;       // [issuing warp]: every product has retired
  uint64_t* turn = fin + 3;         // [softmax warp]: its exponentials of a tile are done
  uint32_t* holder = reinterpret_cast<uint32_t*>(turn + 8);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int s = 0; s < ST; s++) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], C::SW);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int b = 0; b < NB; b++) {
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], 4);
      mbar_init(&o_done[b], 1);
    }
    for (int w = 0; w < 2; w++) mbar_init(&q_full[w], 1);
    for (int k = 0; k < 3; k++) mbar_init(&fin[k], 1);
    for (int k = 0; k < 8; k++) mbar_init(&turn[k], 1);
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
  // Key tiles from the first on. With a bias they begin where the queries are, near their nearest
  // keys, and wrap around: scores that grew from tile to tile on the way there would have the
  // outputs scaled again for each. Both row tiles then take all of them.
  int start = 0;
  if (BIAS) {
    n[0] = rows[0] > 0 ? max(n[0], n[1]) : 0;
    n[1] = rows[1] > 0 ? n[0] : 0;
    start = max(0, min((i0 + D.nk - D.nq) / BN, n[0] - 1));
  }
  auto key_tile = [&](int step) { return start + step < n[0] || !BIAS ? start + step : start + step - n[0]; };
  const int ksteps = (A.head_dim + 15) / 16;

  // registers: 384 threads begin with 168 each; the softmax groups take what the third gives
  // (2 * 128 * 208 + 128 * 80 or 2 * 128 * 216 + 128 * 64, 63488 of 64512; with a bias 200 took 5 %
  // more time, with a cap 208 6 %)
  constexpr int kSoftmaxRegisters = CAP ? 216 : 208, kOtherRegisters = CAP ? 64 : 80;
  if (warp >= 8) {
    fewer_registers<kOtherRegisters>();
    if (warp == 8 && lane == 0) {
      // ------------------------------------------------------------------ loads
      auto load = [&](uint8_t* dst, int bytes, const CUtensorMap* map, uint64_t* bar, int head, int row) {
        mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
        for (int p = 0; p < NP; p++) tma_load_3d(dst + p * (bytes / NP), map, bar, p * 64, head, row);
      };
      const int N = max(n[0], n[1]);
      auto bar = [&](bool value, int i, bool full) {
        return (full ? value ? v_full : k_full : value ? v_empty : k_empty) + i % ST;
      };
      load_tiles<ST>(
          N, [&](bool value, int i) { return attn_wait(A.launch, bar(value, i, false), ((i / ST) - 1) & 1, DEV_TIMEOUT_EMPTY); },
          [&](bool value, int i) {
            load((value ? vring : kring) + i % ST * C::KB, C::KB, value ? &mapV : &mapK, bar(value, i, true), hk,
                 D.k0 + key_tile(i) * BN);
            if (i == 0 && !value)
              for (int w = 0; w < 2; w++)
                if (n[w] > 0) load(sQ + w * C::QB, C::QB, &mapQ, &q_full[w], h, D.q0 + i0 + w * kTcTile);
          },
          [&](bool value, int i) { wait_landed(bar(value, i, true), (i / ST) & 1); });
      for (int w = 0; w < 2; w++)
        if (n[w] > 0) wait_landed(&q_full[w], 0);
    }
    // values that steer the products, from reductions, which give uniform registers
    const int n0 = (int)__reduce_max_sync(0xffffffffu, (unsigned)n[0]);
    const int n1 = (int)__reduce_max_sync(0xffffffffu, (unsigned)n[1]);
    const int keys = (int)__reduce_max_sync(0xffffffffu, (unsigned)kmax);
    const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
    const int last = max(n0, n1) - 1;
    const int cut = BIAS ? (int)__reduce_max_sync(0xffffffffu, (unsigned)(last - start)) : last;  // step of the last keys
    // after a wait that gave up the products go on without waiting, over whatever is there
    bool ok = true;
    auto wait = [&](uint64_t* bar, int phase, unsigned code) {
      if (ok) ok = attn_wait(A.launch, bar, phase & 1, code);
    };
    if (warp == 9 || (C::SW == 2 && warp == 11)) {
      // ----------------------------------------------------------- score products
      // one warp for both tiles in turn, or one for each
      const int mine = C::SW == 1 ? -1 : warp == 11 ? 1 : 0;
      const uint32_t one = elect_one(), id = idesc_16(128, BN, BF16, false);
      const uint32_t dq = desc_low(smem_u32(sQ), 16), dk = desc_low(smem_u32(kring), 16);
      const int rounds = mine < 0 ? last + 1 : mine ? n1 : n0;
      for (int i = 0, st = 0, ph = 0; i < rounds; i++) {
        wait(&k_full[st], ph, DEV_TIMEOUT_FULL);
#pragma unroll
        for (int x = 0; x < 3 - C::SW; x++) {
          const int w = mine < 0 ? x : mine;
          if (i < (w ? n1 : n0)) {
            const Place at(w, i, n0, n1);
            if (i == 0) wait(&q_full[w], 0, DEV_TIMEOUT_FULL);
            // the output product of the buffer's last use (at first there is none: the parity
            // is then that of the phase before)
            wait(&o_done[at.buffer], at.parity ^ 1, DEV_TIMEOUT_ACC);
            __syncwarp();
            tc_fence_after();
            const uint32_t q = dq + w * (C::QB >> 4), k = dk + st * (C::KB >> 4), d = tm + at.buffer * BN;
            if (one) {
              mma_ss<false>(d, q, k, id);
#pragma unroll
              for (int c = 1; c < 4 * NP; c++)
                if (c < ksteps)
                  mma_ss<true>(d, q + (((c >> 2) * kTcTile * 128 + (c & 3) * 32) >> 4),
                               k + (((c >> 2) * BN * 128 + (c & 3) * 32) >> 4), id);
              tc_commit(&s_full[at.buffer]);
            }
            __syncwarp();
          }
        }
        if (one) {
          tc_commit(&k_empty[st]);
          // for the other tile's warp, if that tile does not need this one
          if (C::SW == 2 && i >= (mine ? n0 : n1)) tc_commit(&k_empty[st]);
        }
        __syncwarp();
        if (++st == ST) {
          st = 0;
          ph ^= 1;
        }
      }
      if (one) tc_commit(&fin[mine == 1]);
      __syncwarp();
      attn_wait(A.launch, &fin[mine == 1], 0, DEV_TIMEOUT_ACC);
    } else if (warp == 10) {
      // ---------------------------------------------------------- output products
      // V is read along its rows as the contraction (keys contract, values are the N extent):
      // panels of 64 values BN * 128 bytes apart
      const uint32_t one = elect_one(), id = idesc_16(128, ksteps * 16, BF16, true);
      const uint32_t dv = desc_low(smem_u32(vring), BN * 128);
      for (int i = 0, st = 0, ph = 0; i <= last; i++) {
        const int tail = keys - last * BN, steps = (tail + 15) / 16;
        wait(&v_full[st], ph, DEV_TIMEOUT_FULL);
        if (i == cut && tail % 16) {
          // Keys that no row sees, and rows of other documents behind them, have zero weights:
          // what lies there must not reach the product, which takes keys by 16.
          for (int x = 0; x < NP; x++)
            for (int c = tail * 8 + lane; c < steps * 16 * 8; c += 32)
              *reinterpret_cast<uint4*>(vring + st * C::KB + x * BN * 128 + c * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
        }
        const uint32_t v = dv + st * (C::KB >> 4);
#pragma unroll
        for (int w = 0; w < 2; w++)
          if (i < (w ? n1 : n0)) {
            const Place at(w, i, n0, n1);
            wait(&p_full[at.buffer], at.parity, DEV_TIMEOUT_ACC);
            __syncwarp();
            tc_fence_after();
            const uint32_t d = tm + C::OUT + w * 64 * NP, p = tm + at.buffer * BN;
            if (one) {
              mma_ts(d, p, v, id, i != 0);
              if (i != cut) {
#pragma unroll
                for (int c = 1; c < BN / 16; c++) mma_ts(d, p + c * 8, v + c * (2048 >> 4), id);
              } else {
                for (int c = 1; c < steps; c++) mma_ts(d, p + c * 8, v + c * (2048 >> 4), id);
              }
              tc_commit(&o_done[at.buffer]);
            }
            __syncwarp();
          }
        if (one) tc_commit(&v_empty[st]);
        __syncwarp();
        if (++st == ST) {
          st = 0;
          ph ^= 1;
        }
      }
      if (one) tc_commit(&fin[2]);
      __syncwarp();
      attn_wait(A.launch, &fin[2], 0, DEV_TIMEOUT_ACC);
    }
  } else {
    more_registers<kSoftmaxRegisters>();
    // ------------------------------------------------------------------ softmax
    const int w = warp >> 2, r = tid & 127;
    const int rows_w = w ? rows[1] : rows[0], n_w = w ? n[1] : n[0];
    const int first = i0 + w * kTcTile;       // the tile's first query
    const int i = first + r;                  // this thread's query
    const bool live = r < rows_w;
    const int mine = live ? seen(A, D, i) : 0;
    const int open = rows_w > 0 ? seen(A, D, first) : 0;  // keys that every row sees
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t to = lanes + C::OUT + w * 64 * NP;
    const float unit = A.scale * kLog2e, raw_cap = A.cap / A.scale;
    const float to_cap = A.cap > 0.0f ? A.scale / A.cap : 0.0f;
    const F2 unit2 = f2_both(unit);
    // after a wait that gave up the group goes on without waiting, so that its four warps still
    // meet at their barrier
    bool ok = true;
    float m = -INFINITY, l = 0.0f;
    auto output_done = [&](int t) {
      const Place at(w, t, n[0], n[1]);
      if (ok) ok = attn_wait(A.launch, &o_done[at.buffer], at.parity, DEV_TIMEOUT_ACC);
      __syncwarp();
      tc_fence_after();
    };
    // the outputs of this warp's rows so far, times `keep` (the lane's row)
    auto scale_outputs = [&](int t, float keep) {
      output_done(t - 1);  // this tile's waits for the weights
      for (int c = 0; c < ksteps * 16; c += 16) {
        uint32_t o[16];
        tmem_ld16(to + c, o);
#pragma unroll
        for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
        tmem_st16(to + c, o);
      }
    };
    // With a bias the two softmax warps of a scheduler (warp and warp ^ 4) take turns at the
    // exponentials, so that one's keep the special function unit busy while the other is at its
    // bias (12 heads of 64, six images of up to 4096 tokens: 338 -> 308 us when they were added,
    // 290 now; without a bias turns cost more than they give, 193 -> 238 us at 37
    // heads of 64 x 4096^2).
    auto my_turn = [&](int t) {
      const int u = w ? t : t - 1;  // tile 0 first
      if (ok && u >= 0 && u < (w ? n[0] : n[1])) ok = attn_wait(A.launch, &turn[warp ^ 4], u & 1, DEV_TIMEOUT_ACC);
      __syncwarp();
    };
    auto turn_over = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(&turn[warp]);
    };
    auto weights_done = [&](int b) {
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[b]);
    };

    if constexpr (!BIAS) {
      // a row a thread
      float base = 0.0f;  // of the exponents
      bool some_large = false;
      auto new_base = [&]() {
        const float b = m == -INFINITY ? 0.0f : m * unit;
        const bool large = MODE != 1 && fabsf(b) >= kLargeScore;
        base = kTcLift<T> - (large ? 0.0f : b);
        if (MODE != 1) some_large = __any_sync(0xffffffffu, large);
      };
      // Tiles from t on, until all are done or, where rows with large maxima are not taken, the first
      // such row; that tile is begun again (its scores are still there). A loop of its own: as a branch
      // in one loop for all it cost 511 -> 566 us (causal 16384 back to back), as two loops 519.
      auto walk = [&](auto form, int t) {
        constexpr bool LARGE = decltype(form)::value;
        for (; t < n_w; t++) {
          const Place at(w, t, n[0], n[1]);
          const uint32_t ts = lanes + at.buffer * BN;
          if (ok) ok = attn_wait(A.launch, &s_full[at.buffer], at.parity, DEV_TIMEOUT_ACC);
          __syncwarp();
          tc_fence_after();
          uint32_t raw[BN / 32][32];
#pragma unroll
          for (int c = 0; c < BN / 32; c++) tmem_ld32_nw(ts + c * 32, raw[c]);
          tc_wait_ld();
#pragma unroll
          for (int c = 0; c < BN / 32; c++) loaded(raw[c]);
          float(&s)[BN] = reinterpret_cast<float(&)[BN]>(raw);
          if constexpr (CAP) capped(s, to_cap, raw_cap);
          if ((t + 1) * BN > open) {
            const int last = mine - t * BN;
#pragma unroll
            for (int j = 0; j < BN; j++)
              if (j >= last) s[j] = -INFINITY;
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < BN; j += 2) top[(j >> 1) & 3] = max3(top[(j >> 1) & 3], s[j], s[j + 1]);
          const float high = fmaxf(max3(top[0], top[1], top[2]), top[3]);
          if (t == 0) {
            m = high;
            new_base();
            if (!LARGE && some_large) return t;
          } else if (__any_sync(0xffffffffu, (high - m) * unit > 8.0f)) {
            const float next = fmaxf(m, high), keep = next == -INFINITY ? 1.0f : ex2(growth(m, next, unit));
            m = next;
            l *= keep;
            new_base();
            scale_outputs(t, keep);
            if (!LARGE && some_large) return t;
          }
          if constexpr (LARGE) {
            const F2 shift = f2_both(base == kTcLift<T> && m != -INFINITY ? -m : 0.0f);
#pragma unroll
            for (int j = 0; j < BN; j += 2) {
              const float2 x = f2_unpack(f2_add(f2_pack(s[j], s[j + 1]), shift));
              s[j] = x.x;
              s[j + 1] = x.y;
            }
          }
          const F2 base2 = f2_both(base);
          F2 sum[2] = {0, 0};  // two zeros each
#pragma unroll
          for (int c = 0; c < BN / 64; c++) {
            uint32_t p[32];
#pragma unroll
            for (int j = 0; j < 32; j++) {
              const float2 x = f2_unpack(f2_fma(f2_pack(s[64 * c + 2 * j], s[64 * c + 2 * j + 1]), unit2, base2));
              const float2 y = make_float2(ex2(x.x), ex2(x.y));
              sum[j & 1] = f2_add(sum[j & 1], f2_pack(y.x, y.y));
              p[j] = pack2<T>(y.x, y.y);
            }
            tmem_st32_nw(ts + c * 32, p);
          }
          const float2 total = f2_unpack(f2_add(sum[0], sum[1]));
          l += total.x + total.y;
          weights_done(at.buffer);
        }
        return t;
      };
      const int from = walk(std::false_type(), 0);
      if constexpr (MODE != 1)
        if (__builtin_expect(from < n_w, 0)) walk(std::true_type(), from);
    } else {
      // Four rows a thread, g + 8 R, and of each eight keys the two of the lane's place in its quad:
      // a key's positions then serve four scores. (With a row a thread every thread read all the
      // tile's positions, and shared memory was what bound it.)
      const int g = lane >> 2, t4 = lane & 3;
      float rm[4], rl[4], qf[4][NA];
      int rseen[4], ref[NA], kraw[NA];
      float* pos = spos + w * 2 * S2S_MAX_AXES * BN;
      // The bias as slope (|d| + sum of other axes' |ratio d|), the axis with the largest slope first:
      // distances come from the positions' differences, exact where both are near the tile's first
      // query, and each further axis costs two packed operations and an absolute addition. (As
      // |slope q - slope k| neighbours would be off by the rounding of products that grow along the
      // tile; the difference times each axis' slope took 333 us for the six images where this took 303.)
      int axis[NA];
      float slope = 0.0f, ratio[NA];
#pragma unroll
      for (int a = 0; a < NA; a++) axis[a] = a;
#pragma unroll
      for (int a = 0; a < NA; a++)
        if (n_w > 0) {
          ratio[a] = fabsf(A.slopes[a * A.q_heads + h]);
          if (!(ratio[a] <= slope)) {
            if (a > 0) {
              ratio[a] = slope;
              axis[a] = axis[0];
              axis[0] = a;
            }
            slope = fabsf(A.slopes[a * A.q_heads + h]);
          }
        }
#pragma unroll
      for (int a = 1; a < NA; a++) ratio[a] = slope > 0.0f ? ratio[a] / slope : slope;
      slope /= A.scale;
      // the positions of a tile's keys, each loaded a tile ahead by one thread
      auto key_positions = [&](int t) {
        const int j = key_tile(t) * BN + r;
        if (r < BN)
#pragma unroll
          for (int a = 0; a < NA; a++)
            kraw[a] = j < D.nk ? A.kpos[(int64_t)axis[a] * A.kv_tokens + D.k0 + j] : ref[a];
      };
#pragma unroll
      for (int R = 0; R < 4; R++) {
        const int x = (warp & 3) * 32 + g + 8 * R;
        rm[R] = -INFINITY;
        rl[R] = 0.0f;
        rseen[R] = x < rows_w ? seen(A, D, first + x) : 0;
      }
      if (n_w > 0) {
#pragma unroll
        for (int a = 0; a < NA; a++) {
          const int* qa = A.qpos + (int64_t)axis[a] * A.q_tokens + D.q0;
          ref[a] = qa[i0];
#pragma unroll
          for (int R = 0; R < 4; R++) {
            const int x = (warp & 3) * 32 + g + 8 * R;
            qf[R][a] = -(float)(int)((unsigned)qa[x < rows_w ? first + x : i0] - (unsigned)ref[a]);
          }
        }
        key_positions(0);
      }
      bool some_large = false;
      auto look_for_large = [&]() {
        bool large = false;
#pragma unroll
        for (int R = 0; R < 4; R++) large = large || (rm[R] != -INFINITY && fabsf(rm[R] * unit) >= kLargeScore);
        some_large = __any_sync(0xffffffffu, large);
      };
      auto walk = [&](auto form, const int from) {  // as above
        constexpr bool LARGE = decltype(form)::value;
        int t = from;
        for (; t < n_w; t++) {
          const Place at(w, t, n[0], n[1]);
          const uint32_t ts = lanes + at.buffer * BN;
          float* kp = pos + (t & 1) * S2S_MAX_AXES * BN;
          if (!LARGE || t > from) {  // of a tile that is begun again they are there
            if (r < BN)
#pragma unroll
              for (int a = 0; a < NA; a++)
                kp[a * BN + r] = (float)(int)((unsigned)kraw[a] - (unsigned)ref[a]);
            group_sync(1 + w);
            if (t + 1 < n_w) key_positions(t + 1);
          }
          if (ok) ok = attn_wait(A.launch, &s_full[at.buffer], at.parity, DEV_TIMEOUT_ACC);
          __syncwarp();
          tc_fence_after();
          // [half][64 keys]: value 4 k + e is key 8 k + 2 t4 + (e & 1) of row R = 2 half + (e >> 1)
          uint32_t raw[2][BN / 64][32];
#pragma unroll
          for (int x = 0; x < 2; x++)
#pragma unroll
            for (int c = 0; c < BN / 64; c++) tmem_ld_frag(ts + ((uint32_t)x << 20) + c * 64, raw[x][c]);
          tc_wait_ld();
#pragma unroll
          for (int x = 0; x < 2; x++)
#pragma unroll
            for (int c = 0; c < BN / 64; c++) loaded(raw[x][c]);
          float(&s)[2][BN / 64][32] = reinterpret_cast<float(&)[2][BN / 64][32]>(raw);
          if (A.cap > 0.0f) capped(reinterpret_cast<float(&)[BN]>(raw), to_cap, raw_cap);
          const F2 by = f2_both(NA > 1 ? -slope : slope);
#pragma unroll
          for (int c = 0; c < BN / 64; c++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
              F2 k2[NA];
#pragma unroll
              for (int a = 0; a < NA; a++)
                k2[a] = *reinterpret_cast<const F2*>(kp + a * BN + 64 * c + 8 * k + 2 * t4);
#pragma unroll
              for (int R = 0; R < 4; R++) {
                float* x = &s[R >> 1][c][4 * k + 2 * (R & 1)];
                if constexpr (NA == 1) {
                  const float2 d = f2_unpack(f2_mul(f2_add(k2[0], f2_both(qf[R][0])), by));
                  const float2 e = f2_unpack(f2_add(f2_pack(x[0], x[1]), f2_pack(-fabsf(d.x), -fabsf(d.y))));
                  x[0] = e.x;
                  x[1] = e.y;
                } else {
                  float2 d = f2_unpack(f2_add(k2[0], f2_both(qf[R][0])));
#pragma unroll
                  for (int a = 1; a < NA; a++) {
                    const float2 y = f2_unpack(f2_mul(f2_add(k2[a], f2_both(qf[R][a])), f2_both(ratio[a])));
                    d.x = fabsf(d.x) + fabsf(y.x);
                    d.y = fabsf(d.y) + fabsf(y.y);
                  }
                  const float2 z = f2_unpack(f2_fma(f2_pack(d.x, d.y), by, f2_pack(x[0], x[1])));
                  x[0] = z.x;
                  x[1] = z.y;
                }
              }
            }
          if ((key_tile(t) + 1) * BN > open) {
            const int j0 = key_tile(t) * BN + 2 * t4;
#pragma unroll
            for (int c = 0; c < BN / 64; c++)
#pragma unroll
              for (int k = 0; k < 8; k++)
#pragma unroll
                for (int R = 0; R < 4; R++)
#pragma unroll
                  for (int e = 0; e < 2; e++)
                    if (j0 + 64 * c + 8 * k + e >= rseen[R]) s[R >> 1][c][4 * k + 2 * (R & 1) + e] = -INFINITY;
          }
          float high[4];
          bool more = false;
#pragma unroll
          for (int R = 0; R < 4; R++) {
            float x = -INFINITY;
#pragma unroll
            for (int c = 0; c < BN / 64; c++)
#pragma unroll
              for (int k = 0; k < 8; k++)
                x = max3(x, s[R >> 1][c][4 * k + 2 * (R & 1)], s[R >> 1][c][4 * k + 2 * (R & 1) + 1]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            high[R] = x;
            if (t == 0) rm[R] = high[R];
            more = more || (high[R] - rm[R]) * unit > 8.0f;
          }
          if (t == 0) {
            look_for_large();
            if (!LARGE && some_large) return t;
          } else if (__any_sync(0xffffffffu, more)) {
            float keep[4], mine4 = 1.0f;
#pragma unroll
            for (int R = 0; R < 4; R++) {
              const float next = fmaxf(rm[R], high[R]);
              keep[R] = next == -INFINITY ? 1.0f : ex2(growth(rm[R], next, unit));
              rm[R] = next;
              rl[R] *= keep[R];
              const float x = __shfl_sync(0xffffffffu, keep[R], (lane & 7) * 4);
              if (lane >> 3 == R) mine4 = x;
            }
            look_for_large();
            scale_outputs(t, mine4);
            if (!LARGE && some_large) return t;
          }
          F2 base2[4], sum[4];
#pragma unroll
          for (int R = 0; R < 4; R++) {
            const float b = rm[R] == -INFINITY ? 0.0f : rm[R] * unit;
            base2[R] = f2_both(kTcLift<T> - b);
            sum[R] = 0;  // two zeros
            if constexpr (LARGE)
              if (fabsf(b) >= kLargeScore) {
                base2[R] = f2_both(kTcLift<T>);
#pragma unroll
                for (int c = 0; c < BN / 64; c++)
#pragma unroll
                  for (int k = 0; k < 8; k++)
#pragma unroll
                    for (int e = 0; e < 2; e++) s[R >> 1][c][4 * k + 2 * (R & 1) + e] -= rm[R];
              }
          }
          my_turn(t);
#pragma unroll
          for (int x = 0; x < 2; x++)
#pragma unroll
            for (int c = 0; c < BN / 64; c++) {
              uint32_t p[16];
#pragma unroll
              for (int k = 0; k < 16; k++) {
                const int R = 2 * x + (k & 1);
                const float2 z = f2_unpack(f2_fma(f2_pack(s[x][c][2 * k], s[x][c][2 * k + 1]), unit2, base2[R]));
                const float2 y = make_float2(ex2(z.x), ex2(z.y));
                sum[R] = f2_add(sum[R], f2_pack(y.x, y.y));
                p[k] = pack2<T>(y.x, y.y);
              }
              tmem_st_frag(ts + ((uint32_t)x << 20) + c * 32, p);
            }
#pragma unroll
          for (int R = 0; R < 4; R++) {
            const float2 total = f2_unpack(sum[R]);
            rl[R] += total.x + total.y;
          }
          turn_over();
          weights_done(at.buffer);
        }
        return t;
      };
      const int from = walk(std::false_type(), 0);
      if (__builtin_expect(from < n_w, 0)) walk(std::true_type(), from);
      // to the row of the lane
#pragma unroll
      for (int R = 0; R < 4; R++) {
        rl[R] += __shfl_xor_sync(0xffffffffu, rl[R], 1);
        rl[R] += __shfl_xor_sync(0xffffffffu, rl[R], 2);
        const float x = __shfl_sync(0xffffffffu, rm[R], (lane & 7) * 4);
        const float y = __shfl_sync(0xffffffffu, rl[R], (lane & 7) * 4);
        if (lane >> 3 == R) {
          m = x;
          l = y;
        }
      }
    }

    // ------------------------------------------------------------------- output
    if (n_w > 0) output_done(n_w - 1);
    const bool none = m == -INFINITY && l == 0.0f;  // a sum that is NaN is kept
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
      A.lse[(int64_t)h * A.q_tokens + D.q0 + i] = none ? -INFINITY : log_sum<(int)kTcLift<T>>(m, unit, l);
    // keys of the document that this row does not see had zero weights: a NaN or infinity among
    // their values shows here
    unsigned redo = __ballot_sync(0xffffffffu, check != 0.0f && live && mine < kmax);
    __syncwarp();
    while (redo) {
      const int src = __ffs(redo) - 1;
      redo &= redo - 1;
      attend_row<T>(A, D, first + (warp & 3) * 32 + src, h, kmax, lane);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

template <typename T, int NP, int MODE>
cudaError_t launch_attention_tc(AttnArgs& A, cudaStream_t st) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  using C = TcCfg<NP>;
  auto kernel = k_attention_tc<T, NP, MODE>;
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

template <typename T, int NP>
cudaError_t launch_attention_tc(AttnArgs& A, cudaStream_t st) {
  return A.axes > 2                     ? launch_attention_tc<T, NP, 4>(A, st)
         : A.axes > 1                   ? launch_attention_tc<T, NP, 3>(A, st)
         : A.axes                       ? launch_attention_tc<T, NP, 2>(A, st)
         : A.cap == 0.0f                ? launch_attention_tc<T, NP, 0>(A, st)
         : A.cap * kLog2e < kLargeScore ? launch_attention_tc<T, NP, 1>(A, st)
                                        : launch_attention_tc<T, NP, 5>(A, st);
}

template <typename T>
cudaError_t launch_attention_tc(AttnArgs& A, cudaStream_t st) {
  return A.head_dim <= 64 ? launch_attention_tc<T, 1>(A, st) : launch_attention_tc<T, 2>(A, st);
}

}  // namespace
}  // namespace s2s
