// Paged attention for wide tiles (17 to 256 query-head rows) over 8-bit or 16-bit caches,
// with a causal limit, a window and sinks, on the 5th-generation tensor cores.
//
// One CTA = one item of be_paged_plan x one KV head: two row tiles of 128 (row r of the
// item is query r / g, head r % g, so a KV head's tokens are loaded once for its g
// query heads) against steps of 128 tokens, in one pass with a running maximum:
//   * loader warps (4; with 8 the registers of the softmax run short, 8-bit prompts 4 % slower): tokens'
//     rows by cp.async into the canonical 128-byte swizzle, 8-bit codes into the place of
//     their own row, where the same warp spreads them into halves; tokens are addressed one by
//     one, so any page size and the joint of sinks and window cost nothing;
//   * a warp per row tile issues S = Q K^T (128 x 64 x D) into TMEM and O += P V (128 x D x 64) with
//     P read from TMEM, in halves of a step (one warp for both tiles spent 2 560 clocks a half, most
//     of them between its own waits): a row tile has two buffers of S, so the scores of the next
//     half are there when its softmax comes to them.  (128 x 128 products with one buffer
//     left the softmax waiting for P V and S of its own tile, 1 560 of 4 270 clocks a step;
//     128 x 64 x 16 takes 49 clocks instead of 32, bound by shared memory, 128 x 128 x 16 takes 65.)
//   * softmax warps (8 per row tile, two threads per row with 32 scores of a half each): scores from
//     TMEM to registers, maximum, P written over the thread's own scores; P of a half goes out
//     while the next scores come in.  O is rescaled only when a row's maximum grows by more than
//     2^8, so the two threads of a row only agree that it did not (a barrier of their two
//     warps, with a vote); their sums meet at the end.  One thread per row left a third of the
//     issue slots used, two softmax warps per scheduler in a chain of dependent steps.
//     The loops stay short because 22 warps in three roles share the instruction cache: with 128
//     scores per pass and every variant unrolled, fetching instructions took half of each step.
// TMEM: S/P of tile 0 (two buffers of 64) | of tile 1 | O of tile 0 | O of tile 1 = 256 + 2 D columns
// (512 allocated).  S of half j + 2 overwrites P of half j: both products come from one thread,
// and the tensor core runs them in the order of issue.
//
// 8-bit caches: as in the narrow kernel the codes become halves by one exact conversion.  s_K multiplies
// the score.  s_V = 2^E mu with mu in [1, 2): the loaders multiply V's halves by 2^(E - u), u the largest E of
// the first step's tokens, which is exact from 2^-15 (codes down to 2^-9, fp16 down to 2^-24) to 2^7
// (448 * 2^7 = 57 344), and log2 mu joins the exponent.  P then has fp16's range to itself (2^-24 to
// 2^15), whatever the scales of other pages are.  Values of tokens outside those 23 binary orders are 0
// in that pass over the item's tokens, and where one has a code that is not 0 the item is walked again for it: a pass
// per 23 orders, from the lowest up (O times 2^-23 per window in between), with the maximum and
// sum of the first.  (log2 s_V as a whole in the exponent would need no pass, but a page whose scale is
// 2^25 above the others' takes their factors below fp16's smallest.)  A group of
// 8 tokens of one page costs one shared-memory read and three operations per row.  The
// planner aligns ranges to 8 tokens; pages that are no multiple of 8 take scales token by token.
//
// Measured: bf16, 8192 tokens, 32 heads on 8, window 1024 + 4: 227 us, 570 TFLOP/s; 8-bit cache, a
// prompt of 4096 tokens, causal: 213 us, 646 TFLOP/s (209 before V's halves were scaled).  A half
// takes 2 500 clocks per CTA against 1 280 of the tensor core and 1 024 of the exponentials: the rest is the latency of the softmax's steps
// (scores out of TMEM 500, exponentials 1 100 while four warps share a scheduler's unit).
//
// Values that are not finite: 0 * NaN is NaN in the product, so in steps that some row
// sees in part the loaders replace them by 0 and the rows that see them mark
// the dims in shared memory (+inf, -inf, or both for NaN), applied to O at the end.
//
// Every wait is bounded (2 s); one that runs out sets the device status and the abort flag, and all
// roles leave their loops.
#include <climits>

#include "common.cuh"

namespace be {

constexpr int PW_TOK = 128;                    // tokens per step
constexpr int PW_SOFT = 16, PW_LOADERS = 4;    // softmax warps, loader warps; and 2 issuers
constexpr int PW_THREADS = (PW_SOFT + PW_LOADERS + 2) * 32;
constexpr int PW_HALF = PW_TOK * 128;          // 64 dims of 128 rows
constexpr int PW_STAGES = 2;
// exponents of V scales that one pass serves, relative to its unit
constexpr int PW_LOW = -15, PW_SPAN = 23;

template <int D>
struct PwSmem {
  static constexpr int TILE = (D / 64) * PW_HALF;      // one 128 x D operand tile
  static constexpr int Q = 0, K = 2 * TILE, V = K + PW_STAGES * TILE, ODD = V + PW_STAGES * TILE;
  static constexpr int TAB = ODD + 256 * (D / 32) * 8;  // two bit masks of D dims per row
  static constexpr int RS = TAB + 4 * PW_TOK * 16;      // scales of 4 steps' tokens
  static constexpr int MX = RS + 256 * 4;               // scales of the rows
  static constexpr int BAR = MX + 2 * 256 * 4;          // the threads' maxima, then sums
  static constexpr int BYTES = BAR + 256 + 1024;        // (32 slots of 8 bytes; the alignment)
};

// The elected lane's 1; whole warps call these.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r;
}
// D[tmem] (+)= A[smem] * B[smem] and D[tmem] (+)= A[tmem] * B[smem], kind::f16
__device__ __forceinline__ void umma_f16_el(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc,
                                            uint32_t accumulate, uint32_t el) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(el)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ts_el(uint32_t tmem_d, uint32_t tmem_a, uint64_t b,
                                               uint32_t idesc, uint32_t accumulate, uint32_t el) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(b), "r"(idesc), "r"(accumulate), "r"(el)
      : "memory");
}
__device__ __forceinline__ void umma_commit_el(uint64_t* bar, uint32_t el) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(
          smem_u32(bar)), "r"(el)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// two fp32 operations in one instruction (sm_100)
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint32_t low_bits(int n) {         // bits [0, n), n clamped to 0 .. 32
  const int k = min(max(n, 0), 32);
  return k == 32 ? ~0u : (1u << k) - 1u;
}
// Barrier `id` of N threads; whether `p` held in one of them.
template <int N>
__device__ __forceinline__ bool vote(int id, bool p) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n"
      " barrier.cta.red.or.pred q, %1, %3, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r) : "r"(id), "r"((uint32_t)p), "n"(N) : "memory");
  return r != 0;
}

__device__ __forceinline__ void tmem_ld16_nw(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// element x of a 16-bit pair: set to zero if not finite
template <typename T>
__device__ __forceinline__ uint32_t zero_not_finite(uint32_t w) {
  const uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  if ((w & e) == e) w &= 0xffff0000u;
  if ((w & (e << 16)) == (e << 16)) w &= 0x0000ffffu;
  return w;
}

// The slow half of a wait, out of line: it would be inlined a dozen times into code that has to fit the
// instruction caches.  The warp sleeps in hardware, up to 20 us at a time: polls without a
// hint come back after some ten clocks, and 24 waiting warps' polls took half of all issue slots.
__device__ __noinline__ bool wait_on(uint64_t* bar, uint32_t parity) {
  uint64_t t0 = 0;
  for (uint32_t n = 1;; ++n) {
    if (mbar_try_sleep(bar, parity, 20000)) return true;
    if ((n & 15) == 0) {
      const uint64_t t = gtimer();
      if (t0 == 0) {
        t0 = t;
      } else if (t - t0 > kWaitNs) {
        atomicCAS(&g_device_status, 0, BE_EDEVICE_TIMEOUT);
        return false;
      }
    }
  }
}

// Bounded wait of a whole warp: every lane sees the phase, and all agree on the outcome.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
  const bool ok = !*abort_flag && wait_on(bar, parity);
  return __all_sync(0xffffffffu, ok);
}

// The same for N threads: one warp polls (`leads`), the others sleep at barrier `id`.
template <int N>
__device__ __forceinline__ bool group_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int id,
                                           bool leads) {
  const bool fail = leads && !warp_wait(bar, parity, abort_flag);
  return !vote<N>(id, fail);
}

template <typename T, typename CT, int D>
__global__ void __launch_bounds__(PW_THREADS, 1) paged_wide_kernel(const PagedParams p) {
  constexpr bool Q8 = std::is_same<CT, E4M3>::value;
  using MT = typename std::conditional<Q8, __half, T>::type;   // type of the products
  using SM = PwSmem<D>;
  constexpr int ROWB = D * CacheElt<CT>::bytes;
  constexpr int CH = ROWB / 16;                 // 16-byte chunks per (token, head) row: 4, 8 or 16
  constexpr int TPI = 32 / CH;                  // tokens per warp and load instruction
  constexpr int UNITS = PW_TOK / TPI;           // such instructions per step, dealt to the warps
  constexpr int NL = PW_LOADERS, ITS = UNITS / NL;
  static_assert(UNITS % NL == 0 && NL * TPI % 8 == 0, "a lane's tokens are the same mod 8");
  static_assert(ITS * TPI <= 32, "a lane locates one token");
  extern __shared__ char smem_raw[];
  // (aligned by an offset, so that the compiler still knows it for shared memory)
  char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::BAR);
  uint64_t* k_full = bars;                      // [2], the loader warps
  uint64_t* v_full = bars + 2;                  // [2]
  uint64_t* k_empty = bars + 4;                 // [2], commit
  uint64_t* v_empty = bars + 6;                 // [2]
  uint64_t* s_full = bars + 8;                  // [row tile][half], commit
  uint64_t* p_full = bars + 12;                 // [row tile][half], 8 softmax warps
  // [row tile][half], commit.  Two P V of a tile can be in flight, so a single barrier's parity could not
  // tell the one waited for from the one before the last.
  uint64_t* o_done = bars + 16;
  uint64_t* drain = bars + 20;                  // [row tile]
  uint64_t* q_full = bars + 27;                 // the softmax warps
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(bars + 22);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 23);
  volatile int* odd = reinterpret_cast<volatile int*>(bars + 24);   // [2] per V stage: step + 1
  volatile int* gone = reinterpret_cast<volatile int*>(bars + 25);  // [4]: step + 1 that misses a page
  volatile int* marked = reinterpret_cast<volatile int*>(bars + 28);   // some row's odd_mask is set
  volatile int* unit = reinterpret_cast<volatile int*>(bars + 29);      // u of the first pass
  volatile uint32_t* needed = reinterpret_cast<volatile uint32_t*>(bars + 30);   // windows: bit 16 + k
  uint32_t* odd_mask = reinterpret_cast<uint32_t*>(smem + SM::ODD);  // [256][2][D / 32]
  // per token of the last 4 steps (the loaders are at most 3 past the softmax, and write a step's
  // entries once V of the third before is used up): s_K, log2 mu, 1 / mu
  float4* tab = reinterpret_cast<float4*>(smem + SM::TAB);
  float* row_scale = reinterpret_cast<float*>(smem + SM::RS);
  float* meet = reinterpret_cast<float*>(smem + SM::MX);             // [2][256]

  pdl_wait();
  const be_paged_plan_info* hdr = reinterpret_cast<const be_paged_plan_info*>(p.plan);
  const int item = blockIdx.x / p.hkv, kvh = blockIdx.x - item * p.hkv;
  // items follow the header, so both are read at once (the plan holds at least one item here)
  const be_paged_item w = reinterpret_cast<const be_paged_item*>(p.plan + BE_PLAN_HEADER_INTS)[item];
  if (item >= hdr->n_work_wide) return;
  const int32_t* kvlist = p.plan + hdr->off_kvlist + w.kv_off;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = p.g, rows = w.q_len * g;
  // row / g for rows below 256 (g <= 128: the error r * 1 / 2^20 stays under 1 / g)
  const int g_inv = (1 << 20) / g + 1;
  auto query_of = [&](int r) { return (r * g_inv) >> 20; };
  const bool two = rows > 128;
  const int steps = (w.v_end - w.v_begin + PW_TOK - 1) / PW_TOK;
  const int halves = (w.v_end - w.v_begin + PW_TOK / 2 - 1) / (PW_TOK / 2);
  const bool causal = (w.flags & BE_ITEM_CAUSAL) != 0, window = w.window >= 0;
  // the last v that a row at `pos` sees, the first past its sinks; with a gap, v >= n0 is t - shift
  auto last_of = [&](int pos) {
    return !causal ? INT_MAX - 1 : w.shift == 0 ? pos : pos >= w.n0 + w.shift ? pos - w.shift : min(pos, w.n0 - 1);
  };
  auto first_of = [&](int pos) {
    return !window ? INT_MIN : w.shift == 0 ? pos - w.window : max(pos - w.window - w.shift, w.n0);
  };
  // whether every row sees every one of the n tokens from v0 (page ids apart)
  const int see_end = min(w.v_end, last_of(w.pos0) + 1);
  const int see_from = first_of(w.pos0 + w.pos_step * (w.q_len - 1));
  auto all_see = [&](int v0, int n) {
    return v0 + n <= see_end && (v0 >= see_from || v0 + n <= w.sink_end);
  };

  // Passes.  Steps count on over them, and so do the phases of the barriers: step i of a pass is
  // done + i; the barriers of even and odd halves start a pass with the phases in bits 0 and 1 of `ph`.
  auto phase = [](int ph, int j) { return ((ph >> (j & 1)) ^ (j >> 1)) & 1; };
  const int ph_step = (steps & 1) | (halves & 2);
  // (no page at all in the first step: any unit)
  auto first_unit = [&]() -> int { return *unit == INT_MIN ? 0 : *unit; };
  // The pass after the one for window k (all roles come to the same: the windows needed are known with
  // the last V tile of a pass): 0 none, 1 for a higher window, 2 for the lowest of all with O begun anew.
  // The first pass is for window 0, whatever the others are; O only ever moves to larger units, where
  // what fp32 loses at its lower end is nothing beside what any token adds.
  auto next_pass = [&](int& k, bool& anew) -> int {
    const uint32_t need = *needed;
    if (!anew && (need & 0xffffu)) {
      anew = true;
      k = __ffs(need) - 17;
      return 2;
    }
    const uint32_t up = (need | (anew ? 1u << 16 : 0u)) & ~((2u << (k + 16)) - 1u);
    if (!up) return 0;
    k = __ffs(up) - 17;
    return 1;
  };

  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], NL);
      mbar_init(&v_full[s], NL);
      mbar_init(&k_empty[s], two ? 2 : 1);      // a commit per row tile
      mbar_init(&v_empty[s], two ? 2 : 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&o_done[2 * s + h], 1);
        mbar_init(&s_full[2 * s + h], 1);
        mbar_init(&p_full[2 * s + h], PW_SOFT / 2);
      }
      odd[s] = gone[s] = gone[2 + s] = 0;
    }
    mbar_init(drain, 1);
    mbar_init(q_full, PW_SOFT);
    mbar_init(drain + 1, 1);
    *abort_flag = 0;
    *marked = 0;
    *unit = INT_MIN;
    *needed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32((const void*)tmem_slot)), "n"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= PW_SOFT) {
    if (warp >= PW_SOFT + NL) {
      // ---------------- issuers: a warp for each row tile ----------------
      // The whole warp walks the steps and one elected lane issues: addresses and descriptors
      // then stay in uniform registers (from a divergent lane every product first moves them there)
      const uint32_t el = elect_one();
      const uint32_t id_s = umma_idesc<MT>(128, PW_TOK / 2, 0), id_o = umma_idesc<MT>(128, D, 1);
      const uint64_t dq = umma_desc(smem_u32(smem + SM::Q), 16, 1024);
      const uint64_t dk = umma_desc(smem_u32(smem + SM::K), 16, 1024);
      const uint64_t dv = umma_desc(smem_u32(smem + SM::V), PW_HALF, 1024);
      int done = 0, ph = 0, win = 0;
      bool anew = false, carry = false;
      // half j: tokens [64 (j & 1), + 64) of step j / 2, buffer j & 1 of the tile's S
      auto issue_s = [&](int tile, int j) {
        const uint64_t a = dq + tile * (SM::TILE >> 4);
        const uint64_t b = dk + ((done + (j >> 1)) & 1) * (SM::TILE >> 4) + (j & 1) * (64 * 128 >> 4);
        const uint32_t d = tmem + tile * 128 + (j & 1) * 64;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * PW_HALF + (kk & 3) * 32) >> 4;
          umma_f16_el(d, a + off, b + off, id_s, kk > 0, el);
        }
        umma_commit_el(&s_full[2 * tile + (j & 1)], el);
      };
      auto issue_o = [&](int tile, int j) {
        const uint64_t b = dv + ((done + (j >> 1)) & 1) * (SM::TILE >> 4) + (j & 1) * (4 * 2048 >> 4);
        const uint32_t d = tmem + 256 + tile * D, a = tmem + tile * 128 + (j & 1) * 64;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          umma_f16_ts_el(d, a + (ks >> 1) * 32 + (ks & 1) * 8, b + ks * (2048 >> 4), id_o,
                         ks > 0 || j > 0 || carry, el);
        umma_commit_el(&o_done[2 * tile + (j & 1)], el);
      };
      const int tile = warp - (PW_SOFT + NL);
      const bool idle = tile == 1 && !two;
      bool ok = idle || warp_wait(q_full, 0, abort_flag);
#pragma unroll 1
      while (ok && !idle) {
        ok = warp_wait(&k_full[done & 1], (done >> 1) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        issue_s(tile, 0);
        if (halves > 1) issue_s(tile, 1);
        umma_commit_el(&k_empty[done & 1], el);
#pragma unroll 1
        for (int j = 0; j < halves; ++j) {
          const int i = done + (j >> 1), st = i & 1, nj = j + 2;
          if ((j & 1) == 0) ok = warp_wait(&v_full[st], (i >> 1) & 1, abort_flag);
          if (ok) ok = warp_wait(&p_full[2 * tile + (j & 1)], phase(ph, j), abort_flag);
          if (!ok) break;
          tc_fence_after();
          issue_o(tile, j);
          if ((j & 1) || j + 1 == halves) umma_commit_el(&v_empty[st], el);
          if (nj < halves) {
            const int ni = i + 1;
            if ((nj & 1) == 0) {
              ok = warp_wait(&k_full[ni & 1], (ni >> 1) & 1, abort_flag);
              if (!ok) break;
              tc_fence_after();
            }
            issue_s(tile, nj);
            if ((nj & 1) || nj + 1 == halves) umma_commit_el(&k_empty[ni & 1], el);
          }
        }
        if (!ok || !Q8) break;
        const int next = next_pass(win, anew);
        if (next == 0) break;
        carry = next == 1;
        done += steps;
        ph ^= ph_step;
      }
      if (!ok) {        // leave with no product in flight
        *abort_flag = 1;
        umma_commit_el(drain + tile, el);
        wait_on(drain + tile, 0);
      }
    } else {
      // ---------------- loaders ----------------
      const int lw = warp - PW_SOFT;
      const uint32_t plane = (uint32_t)p.hkv * p.ps;        // rows of ROWB bytes (2^32 of them: 256 GB)
      const char* base = p.pool + (int64_t)kvh * ROWB;
      // Lane: 16-byte chunk c of token `sub`.  Where a row has 8 chunks of codes, the upper 4 lie with the
      // neighbouring token: 8 lanes then store halves without meeting a bank twice.
      const int c = lane % CH, sub = Q8 && CH == 8 ? (lane / CH) ^ (c >> 2) : lane / CH;
      // load instruction `it` of this warp takes tokens [unit * TPI, + TPI), unit = lw + NL it;
      // lane L locates the token that instruction L / TPI loads in place L % TPI
      const int my_tok = (lw + NL * (lane / TPI)) * TPI + lane % TPI;
      const int tok0 = lw * TPI + sub;              // this lane's tokens: tok0 + NL TPI it
      const bool my = lane < ITS * TPI && my_tok < PW_TOK;
      const int ps_shift = (p.ps & (p.ps - 1)) == 0 ? __ffs(p.ps) - 1 : -1;
      auto token_t = [&](int v) { return v + (v >= w.n0 ? w.shift : 0); };
      auto page_of = [&](int v0) -> int {        // page id of this lane's token, -1 past the range
        const int v = v0 + my_tok;
        if (!my || v >= w.v_end) return -1;
        const int t = token_t(v);
        return ld_early4(kvlist + (ps_shift >= 0 ? t >> ps_shift : t / p.ps));
      };
      constexpr uint32_t kNone = ~0u;
      auto locate = [&](int i, int page, float& sk, float& sv) -> uint32_t {
        const int v = w.v_begin + i * PW_TOK + my_tok;
        sk = 0.f;
        sv = -1.f;
        if (page < 0 || page >= p.num_pages) {
          if (my && v < w.v_end) {
            flag_range_error();
            gone[i & 3] = i + 1;                // (16-bit caches look at it: they take one pass)
          }
          return kNone;
        }
        if constexpr (Q8) {
          const float* s = p.scale + (int64_t)page * 2 * p.hkv + kvh;
          sk = ld_early4(s);
          sv = ld_early4(s + p.hkv);
        }
        const int t = token_t(v);
        return (uint32_t)page * 2 * plane +
               (uint32_t)(ps_shift >= 0 ? t & (p.ps - 1) : t % p.ps) * p.hkv;
      };
      auto dst_of = [&](int tok, int chunk) -> uint32_t {   // 16-byte chunk of 8 dims
        return (chunk >> 3) * PW_HALF + tok * 128 + (((chunk & 7) ^ (tok & 7)) << 4);
      };
      auto signal = [&](uint64_t* bar) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
      };
      // Codes land inside the place of their own row (in its last 128 bytes; where they are 64, odd
      // tokens in the second 64: no bank twice) and are spread from there over the whole row by the
      // warp that asked for them.
      // (the offset of a 16-byte chunk is the same for all tokens of a lane but for 128 bytes per token)
      const uint32_t at_raw = Q8 ? (D / 64 - 1) * PW_HALF + tok0 * 128 + ((c + (CH == 4 ? (tok0 & 1) * 4 : 0)) << 4)
                                 : dst_of(tok0, c);
      constexpr uint32_t NEXT = NL * TPI * 128;
      auto copy = [&](char* tile, uint32_t at, uint32_t more) {
        const uint32_t dst = smem_u32(tile) + at_raw;
#pragma unroll
        for (int it = 0; it < ITS; ++it) {
          const uint32_t o = __shfl_sync(0xffffffffu, at, it * TPI + sub);
          cp_async16(dst + it * NEXT, o != kNone ? base + (uint64_t)(o + more) * ROWB + c * 16 : p.pool, o != kNone);
        }
        cp_commit();
      };
      // 8-bit V rows: 2^(E - u) of this lane's token as two halves (0: of another pass) and the bit
      // of its window; of this step and of the one before, whose rows land meanwhile.
      int done = 0, win = 0;
      bool anew = false;
      uint32_t mul = 0, mul_v = 0;
      int bit = 0, bit_v = 0;
      bool some = false, some_v = false;        // a token of the warp's is of another pass
      auto weigh = [&](float sv, bool first) {
        const int e = (int)(__float_as_uint(fmaxf(sv, 9.0949470177e-13f)) >> 23) - 127;      // 2^-40
        const bool has = my && sv >= 0.f;
        if (first) {
          const int top = __reduce_max_sync(0xffffffffu, has ? e : INT_MIN);
          if (lane == 0) atomicMax(const_cast<int*>(unit), top);
          vote<NL * 32>(10, false);
        }
        const int d = has ? e - first_unit() - win * PW_SPAN : 0;
        const bool in = d >= PW_LOW && d < PW_LOW + PW_SPAN;
        mul = !in ? 0u : d < -14 ? 0x02000200u : (uint32_t)(d + 15) * 0x04000400u;
        bit = has ? (e - first_unit() - PW_LOW + 16 * PW_SPAN) / PW_SPAN : 16;
        some = __any_sync(0xffffffffu, !in);
      };
      // Codes of tokens of another pass: 0, and their window asked for where they are not 0.
      auto put_off = [&](char* tile) {
#pragma unroll 1
        for (int it = 0; it < ITS; ++it) {
          const uint32_t h = __shfl_sync(0xffffffffu, mul_v, it * TPI + sub);
          const int b = __shfl_sync(0xffffffffu, bit_v, it * TPI + sub);
          if (h == 0) {
            int4* a = reinterpret_cast<int4*>(tile + at_raw + it * NEXT);
            const int4 x = *a;
            if ((x.x | x.y | x.z | x.w) & 0x7f7f7f7f) atomicOr(const_cast<uint32_t*>(needed), 1u << b);
            *a = make_int4(0, 0, 0, 0);
          }
        }
      };
      // Rows have landed: codes to halves, V's times 2^(E - u); values that are not finite out if `check`.
      const uint32_t at0 = dst_of(tok0, 2 * c), at1 = dst_of(tok0, 2 * c + 1);
      auto finish = [&](char* tile, bool check, bool v) -> bool {
        bool bad = false;
        if constexpr (Q8) {
          constexpr int B = ITS < 2 ? 1 : 2;
#pragma unroll 1
          for (int it = 0; it < ITS; it += B, tile += B * NEXT) {
            int4 raw[B];
#pragma unroll
            for (int u = 0; u < B; ++u) raw[u] = *reinterpret_cast<const int4*>(tile + at_raw + u * NEXT);
            __syncwarp();
#pragma unroll
            for (int u = 0; u < B; ++u) {
              const uint32_t wd[4] = {(uint32_t)raw[u].x, (uint32_t)raw[u].y, (uint32_t)raw[u].z,
                                      (uint32_t)raw[u].w};
              uint32_t o[8];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                o[2 * x] = e4m3x2_to_h2(wd[x] & 0xffffu);
                o[2 * x + 1] = e4m3x2_to_h2(wd[x] >> 16);
              }
              if (v) {
                const uint32_t f = __shfl_sync(0xffffffffu, mul_v, (it + u) * TPI + sub);
#pragma unroll
                for (int x = 0; x < 8; ++x) o[x] = mul_h2(o[x], f);
              }
              if (check) {
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                  const uint32_t z = zero_not_finite<__half>(o[x]);
                  bad |= z != o[x];
                  o[x] = z;
                }
              }
              *reinterpret_cast<int4*>(tile + at0 + u * NEXT) = make_int4(o[0], o[1], o[2], o[3]);
              *reinterpret_cast<int4*>(tile + at1 + u * NEXT) = make_int4(o[4], o[5], o[6], o[7]);
            }
          }
        } else if (check) {
#pragma unroll 1
          for (int it = 0; it < ITS; ++it) {
            int4* a = reinterpret_cast<int4*>(tile + at_raw + it * NEXT);
            const int4 x = *a;
            const int4 z = make_int4(zero_not_finite<T>(x.x), zero_not_finite<T>(x.y),
                                     zero_not_finite<T>(x.z), zero_not_finite<T>(x.w));
            if (z.x != x.x || z.y != x.y || z.z != x.z || z.w != x.w) {
              bad = true;
              *a = z;
            }
          }
        }
        return bad;
      };
      auto finish_v = [&](int i) {        // looked at where rows see the step in part
        char* tile = smem + SM::V + ((done + i) & 1) * SM::TILE;
        if (Q8 && some_v) put_off(tile);
        if (finish(tile, !all_see(w.v_begin + i * PW_TOK, PW_TOK), true))
          odd[(done + i) & 1] = done + i + 1;
        signal(&v_full[(done + i) & 1]);
      };
      bool ok = true;
      float sk, sv;
#pragma unroll 1
      for (;;) {
        int page_next = page_of(w.v_begin);
#pragma unroll 1
        for (int i = 0; i < steps; ++i) {
          const int at_step = done + i, st = at_step & 1, before = ((at_step >> 1) - 1) & 1;
          const uint32_t at = locate(i, page_next, sk, sv);
          page_next = page_of(w.v_begin + (i + 1) * PW_TOK);
          if (at_step >= 2 && !group_wait<NL * 32>(&k_empty[st], before, abort_flag, 10, lw == 0)) {
            ok = false;
            break;
          }
          copy(smem + SM::K + st * SM::TILE, at, 0);
          if constexpr (Q8) {
            mul_v = mul;
            bit_v = bit;
            some_v = some;
            weigh(sv, at_step == 0);
            // scales of 0 (blocks never written) stand for values of 0: any will do; a token that is
            // not there gets an exponent of -inf
            const float mu = __uint_as_float((__float_as_uint(fmaxf(sv, 9.0949470177e-13f)) & 0x7fffffu) | 0x3f800000u);
            if (my)
              tab[(at_step & 3) * PW_TOK + my_tok] =
                  sv < 0.f ? make_float4(1.f, -INFINITY, 0.f, 0.f)
                           : make_float4(fmaxf(sk, 1e-30f), log2f(mu), 1.f / mu, 0.f);
          }
          if (i > 0) {
            cp_wait<1>();
            finish_v(i - 1);
          }
          // K goes out before V's stage is waited for: that one comes free with the step before last
          cp_wait<0>();
          finish(smem + SM::K + st * SM::TILE, false, false);
          signal(&k_full[st]);
          if (at_step >= 2 && !group_wait<NL * 32>(&v_empty[st], before, abort_flag, 10, lw == 0)) {
            ok = false;
            break;
          }
          copy(smem + SM::V + st * SM::TILE, at, plane);
        }
        cp_wait<0>();
        if (!ok) break;
        mul_v = mul;
        bit_v = bit;
        some_v = some;
        finish_v(steps - 1);
        if (!Q8) break;
        vote<NL * 32>(10, false);               // the other warps' windows
        if (next_pass(win, anew) == 0) break;
        done += steps;
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    // ---------------- softmax: two threads per row ----------------
    // ---- Q rows into shared memory, zeros past the item's rows (loads in flight together; one
    // at a time they took 9 us of a CTA's 42 at 18 halves) ----
    {
      constexpr int QC = D / 8, QR = PW_SOFT * 32 / QC, QB = 4;   // chunks per row, rows at once
      // the sign of sm_scale goes into Q, so that the largest score is the largest product
      const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
      const int c = tid % QC;
#pragma unroll 1
      for (int r0 = tid / QC; r0 < (two ? 256 : 128); r0 += QR * QB) {
        int4 v[QB];
#pragma unroll
        for (int k = 0; k < QB; ++k) {
          const int r = r0 + k * QR;
          v[k] = r < rows ? ld_early16(reinterpret_cast<const T*>(p.q) +
                                       (w.q_begin + query_of(r)) * p.q_row_stride +
                                       (int64_t)(kvh * g + r - query_of(r) * g) * D + c * 8)
                          : make_int4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < QB; ++k) {
          const int r = r0 + k * QR;
          uint32_t x[4] = {v[k].x ^ flip, v[k].y ^ flip, v[k].z ^ flip, v[k].w ^ flip};
          if constexpr (Q8) {
            // bf16 rows into half range by a power of two, as in the narrow kernel
            float back = 1.f;
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
              float f[8], mx = 0.f;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x[i]));
                f[2 * i] = y.x;
                f[2 * i + 1] = y.y;
                mx = fmaxf(mx, fmaxf(fabsf(y.x), fabsf(y.y)));
              }
#pragma unroll
              for (int off = QC / 2; off; off >>= 1)
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
              int e = (int)(__float_as_uint(mx) >> 23) - 127;
              e = mx < INFINITY ? min(max(e, -110), 110) : 0;
              const float up = __uint_as_float((uint32_t)(8 - e + 127) << 23);
              back = __uint_as_float((uint32_t)(e - 8 + 127) << 23);
#pragma unroll
              for (int i = 0; i < 4; ++i) x[i] = pack2<__half>(f[2 * i] * up, f[2 * i + 1] * up);
            }
            if (c == 0) row_scale[r] = back;
          }
          *reinterpret_cast<int4*>(smem + SM::Q + (r >> 7) * SM::TILE + (c >> 3) * PW_HALF +
                                   (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4)) =
              make_int4(x[0], x[1], x[2], x[3]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      for (int k = tid; k < 256 * 2 * (D / 32); k += PW_SOFT * 32) odd_mask[k] = 0;
      asm volatile("bar.sync 1, 512;" ::: "memory");           // the rows' scales and masks
      static_assert(PW_SOFT * 32 == 512, "barrier count");
    }
    // rows 0..255 of the item; this thread's scores: tokens [32 part, + 32) of a half
    const int tile = warp >> 3, part = (warp >> 2) & 1, row = tile * 128 + (warp & 3) * 32 + lane;
    if (tile == 0 || two) {
      const uint32_t quad = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t t_s = tmem + tile * 128 + quad, t_o = tmem + 256 + tile * D + quad;
      const int pos = w.pos0 + w.pos_step * query_of(row);
      // factors of scores are never 0: a masked score of -inf stays -inf
      constexpr float kLeast = 1e-37f;
      const float scale = fmaxf(fabsf(p.scale_log2), 1e-30f) * (Q8 ? row_scale[row] : 1.f);
      // groups of 8 tokens lie in one page, or scales go token by token
      const bool by_token = Q8 && !( p.ps % 8 == 0 && w.v_begin % 8 == 0 &&
                           (w.shift == 0 || (w.n0 % 8 == 0 && w.shift % 8 == 0)));
      // what the row sees, in v: v <= vc and (v < sink_end or v >= vw)
      const int vc = last_of(pos), vw = first_of(pos);
      const int pair = 2 + tile * 4 + (warp & 3);     // barrier of the two warps with these rows
      // 8-bit caches: the maximum is taken 2^6 lower, so that P uses fp16 from 2^-24 to 2^15
      // (2^6 for the largest score, 2^8 while its maximum lags behind, 2 for mu)
      constexpr float kHead = Q8 ? 6.f : 0.f;
      float m = kNoMax, l = 0.f;
      // A wait that ran out is told to the warp with the rows' other scores at the barrier of a half, so
      // that both leave their loop at the same place.
      bool fail = false, anew = false;
      int done = 0, ph = 0, win = 0;
      float l_all = 0.f;                              // l of the first pass: the later ones have all of m and l
#pragma unroll 1
      for (;;) {
#pragma unroll 1
        for (int j = 0;; ++j) {
          const int i = done + (j >> 1), v0 = w.v_begin + j * 64 + part * 32;    // step; this thread's tokens
          // this thread's columns: 32 scores, then its P in the first 16 of them
          const uint32_t t_p = t_s + (j & 1) * 64 + part * 32;
          uint32_t x[32];
          if (j < halves) {
            fail = fail || !warp_wait(&s_full[2 * tile + (j & 1)], phase(ph, j), abort_flag);
            tc_fence_after();
            tmem_ld32_nw(t_p, x);
          }
          if (j > 0) {                       // P of the half before goes out while the scores come in
            tmem_wait_st();
            const int i = done + ((j - 1) >> 1), v0 = w.v_begin + (j - 1) * 64 + part * 32;
            if (!all_see(w.v_begin + (i - done) * PW_TOK, PW_TOK)) {
              // values that are not finite, taken out of V: mark the dims of the rows that see them
              // (before P is handed over: V's stage and its flag stay until P V of this half is done)
              fail = fail || !warp_wait(&v_full[i & 1], (i >> 1) & 1, abort_flag);
              if (odd[i & 1] == i + 1) {
                uint32_t* mask = odd_mask + row * (2 * (D / 32));
#pragma unroll 1
                for (int k = 0; row < rows && k < min(32, w.v_end - v0); ++k) {
                  const int v = v0 + k, t = v + (v >= w.n0 ? w.shift : 0);
                  const int page = kvlist[t / p.ps];
                  if (page < 0 || page >= p.num_pages || (causal && t > pos) ||
                      (window && t < pos - w.window && t >= w.sink_end))
                    continue;
                  const int64_t r = ((int64_t)page * 2 + 1) * p.ps + t % p.ps;
                  const char* src = p.pool + (r * p.hkv + kvh) * ROWB;
#pragma unroll 1
                  for (int d = 0; d < D; ++d) {
                    float val;
                    if constexpr (Q8) {
                      const uint32_t h2 = e4m3x2_to_h2(*reinterpret_cast<const uint8_t*>(src + d));
                      val = __low2float(*reinterpret_cast<const __half2*>(&h2));
                    } else {
                      val = to_f(reinterpret_cast<const T*>(src)[d]);
                    }
                    if (!(val < INFINITY)) atomicOr(&mask[d >> 5], 1u << (d & 31));
                    if (!(val > -INFINITY)) atomicOr(&mask[D / 32 + (d >> 5)], 1u << (d & 31));
                  }
                  *marked = 1;
                }
              }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[2 * tile + ((j - 1) & 1)]);
          }
          if (j == halves) break;
          const float4* tb = tab + (i & 3) * PW_TOK + (j & 1) * 64 + part * 32;
          const bool missing = !Q8 && gone[i & 3] == i + 1, cut = !all_see(v0, 32) || missing;
          uint32_t see = ~0u;
          if (cut) {
            const int kc = min(vc >= v0 + 32 ? 32 : vc - v0 + 1, w.v_end - v0);
            const int ks = min(w.sink_end - v0, 32), kw = vw <= v0 ? 0 : min(vw - v0, 32);
            see = low_bits(kc) & (low_bits(ks) | ~low_bits(kw));
            if (missing)                               // a page id out of range: its tokens drop out
#pragma unroll 1
              for (int k = 0; k < min(32, w.v_end - v0); ++k) {
                const int v = v0 + k, t = v + (v >= w.n0 ? w.shift : 0);
                const int page = kvlist[t / p.ps];
                if (page < 0 || page >= p.num_pages) see &= ~(1u << k);
              }
          }
          tmem_wait();
          if (cut) {
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = (see >> k) & 1 ? x[k] : 0xff800000u;             // -inf
          }
          float mx;
          if (by_token) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              x[k] = __float_as_uint(fmaf(__uint_as_float(x[k]), fmaxf(tb[k].x * scale, kLeast), tb[k].y));
          }
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          if (Q8 && !by_token) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              float y[8];
#pragma unroll
              for (int u = 0; u < 8; ++u) y[u] = __uint_as_float(x[k + u]);
              const float gm = fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])),
                                     fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7])));
              m4[k >> 3] = fmaf(gm, fmaxf(tb[k].x * scale, kLeast), tb[k].y);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 32; k += 8)
#pragma unroll
              for (int u = 0; u < 4; ++u)
                m4[u] = fmaxf(fmaxf(m4[u], __uint_as_float(x[k + u])), __uint_as_float(x[k + 4 + u]));
          }
          mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          if (!Q8) mx *= scale;
          if (vote<64>(pair, mx > m + (kHead + kLazyMax) || fail)) {
            meet[part * 256 + row] = mx;
            if (vote<64>(pair, fail)) {
              fail = true;
              break;
            }
            const float to = fmaxf(m, fmaxf(mx, meet[(part ^ 1) * 256 + row]) - kHead), f = ex2(m - to);
            m = to;
            l *= f;
            if (j > 0) {        // O of the halves before: complete, then rescaled, half the dims per thread
              fail = !warp_wait(&o_done[2 * tile + ((j - 1) & 1)], phase(ph, j - 1), abort_flag);
              tc_fence_after();
#pragma unroll 1
              for (int c0 = part * (D / 2); c0 < (part + 1) * (D / 2); c0 += 16) {
                uint32_t y[16];
                tmem_ld16_nw(t_o + c0, y);
                tmem_wait();
#pragma unroll
                for (int k = 0; k < 16; ++k) y[k] = __float_as_uint(__uint_as_float(y[k]) * f);
                tmem_st16(t_o + c0, y);
              }
            }
          }
          // ---- P over S ----
          uint32_t pk[16];
          if (by_token) {
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              const float a = ex2(__uint_as_float(x[k]) - m), b = ex2(__uint_as_float(x[k + 1]) - m);
              l = fmaf(a, tb[k].z, fmaf(b, tb[k + 1].z, l));
              pk[k >> 1] = pack2<MT>(a, b);
            }
          } else {
            const uint64_t s2 = f2_pack(scale, scale), m2 = f2_pack(-m, -m);
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int k0 = 0; k0 < 32; k0 += 8) {
              uint64_t gs = s2, gm = m2;
              float inv = 1.f;
              if constexpr (Q8) {
                const float4 e = tb[k0];
                const float both = fmaxf(e.x * scale, kLeast);
                gs = f2_pack(both, both);
                gm = f2_pack(e.y - m, e.y - m);
                inv = e.z;
                sum[0] = sum[1] = 0;
              }
#pragma unroll
              for (int k = k0; k < k0 + 8; k += 2) {
                const uint64_t y = f2_pack(__uint_as_float(x[k]), __uint_as_float(x[k + 1]));
                float a, b;
                f2_unpack(f2_fma(y, gs, gm), a, b);
                a = ex2(a);
                b = ex2(b);
                sum[(k >> 1) & 1] = f2_add(sum[(k >> 1) & 1], f2_pack(a, b));
                pk[k >> 1] = pack2<MT>(a, b);
              }
              if constexpr (Q8) {
                float a, b;
                f2_unpack(f2_add(sum[0], sum[1]), a, b);
                l = fmaf(a + b, inv, l);
              }
            }
            if constexpr (!Q8) {
              float a, b;
              f2_unpack(f2_add(sum[0], sum[1]), a, b);
              l += a + b;
            }
          }
          tmem_st16(t_p, pk);
        }
        fail = fail || !warp_wait(&o_done[2 * tile + ((halves - 1) & 1)], phase(ph, halves - 1), abort_flag);
        if constexpr (!Q8) break;
        if (vote<64>(pair, fail)) {                     // both warps of the rows go on, or neither
          fail = true;
          break;
        }
        if (done == 0) l_all = l;
        const int was = win, next = next_pass(win, anew);
        if (next == 0) break;
        if (next == 1) {                                // O in the next window's unit
          const float f = __uint_as_float((uint32_t)max(127 - (win - was) * PW_SPAN, 1) << 23);
          tc_fence_after();
#pragma unroll 1
          for (int c0 = part * (D / 2); c0 < (part + 1) * (D / 2); c0 += 16) {
            uint32_t y[16];
            tmem_ld16_nw(t_o + c0, y);
            tmem_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) y[k] = __float_as_uint(__uint_as_float(y[k]) * f);
            tmem_st16(t_o + c0, y);
          }
        }
        done += steps;
        ph ^= ph_step;
      }
      if constexpr (Q8) l = l_all;
      // ---- epilogue: half the dims per thread ----
      meet[part * 256 + row] = l;
      if (!vote<64>(pair, fail)) {
        tc_fence_after();
        l += meet[(part ^ 1) * 256 + row];
        const float inv = (l != 0.f ? 1.f / l : 0.f) * (Q8 ? exp2f((float)(first_unit() + win * PW_SPAN)) : 1.f);
        const bool partial = w.part_base >= 0;
        // through this tile's Q rows (its last product has read them) so that rows leave in whole lines:
        // D / 4 dims of fp32 partials or D / 2 of results at a time, in 4 D bytes per warp and row pair
        constexpr int HD = D / 2, RB = HD * 2;                 // this thread's dims; bytes per row here
        char* mine = smem + SM::Q + tile * SM::TILE + (warp & 7) * 32 * RB;
        constexpr int RC = RB / 16;                            // chunks per row: 8 or 4
#pragma unroll 1
        for (int h = 0; h < (partial ? 2 : 1); ++h) {
          const int d0 = part * HD + (partial ? h * (HD / 2) : 0), nd = partial ? HD / 2 : HD;
#pragma unroll 1
          for (int c0 = 0; c0 < nd; c0 += 16) {
            uint32_t u[16];
            tmem_ld16_nw(t_o + d0 + c0, u);
            tmem_wait();
            float f[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) f[k] = l != 0.f ? __uint_as_float(u[k]) * inv : 0.f;
            if (*marked) {
              const int d = d0 + c0;
              const uint32_t up = odd_mask[row * (2 * (D / 32)) + (d >> 5)] >> (d & 31);
              const uint32_t dn = odd_mask[row * (2 * (D / 32)) + D / 32 + (d >> 5)] >> (d & 31);
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                if ((up >> k) & 1) f[k] += INFINITY;
                if ((dn >> k) & 1) f[k] -= INFINITY;
              }
            }
            // 16-byte chunks, turned by the row so that neither side meets a bank twice
            if (partial) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                *reinterpret_cast<float4*>(mine + lane * RB + (((c0 / 4 + k) ^ (lane & (RC - 1))) << 4)) =
                    make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
            } else {
#pragma unroll
              for (int k = 0; k < 2; ++k)
                *reinterpret_cast<uint4*>(mine + lane * RB + (((c0 / 8 + k) ^ (lane & (RC - 1))) << 4)) =
                    make_uint4(pack2<T>(f[8 * k], f[8 * k + 1]), pack2<T>(f[8 * k + 2], f[8 * k + 3]),
                               pack2<T>(f[8 * k + 4], f[8 * k + 5]), pack2<T>(f[8 * k + 6], f[8 * k + 7]));
            }
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < RC; ++k) {
            const int at = lane + 32 * k, rr = at / RC, ch = at % RC;
            const int ir = tile * 128 + (warp & 3) * 32 + rr;
            if (ir >= rows) continue;
            const uint4 val = *reinterpret_cast<const uint4*>(mine + rr * RB + ((ch ^ (rr & (RC - 1))) << 4));
            const int iq = query_of(ir), ih = kvh * g + ir - iq * g;
            if (partial)
              *reinterpret_cast<uint4*>(p.mid_o + ((int64_t)(w.part_base + iq) * p.hq + ih) * D + d0 +
                                        ch * 4) = val;
            else {
              T* dst = reinterpret_cast<T*>(p.out) + (int64_t)(w.q_begin + iq) * p.out_row_stride +
                       (int64_t)ih * D + d0 + ch * 8;
              if (p.out_vec16) *reinterpret_cast<uint4*>(dst) = val;
              else {
                reinterpret_cast<uint2*>(dst)[0] = make_uint2(val.x, val.y);
                reinterpret_cast<uint2*>(dst)[1] = make_uint2(val.z, val.w);
              }
            }
          }
          __syncwarp();
        }
        if (row < rows && part == 0) {
          const int qi = query_of(row), head = kvh * g + row - qi * g;
          const int64_t dst_q = partial ? w.part_base + qi : w.q_begin + qi;
          const float lse = l > 0.f ? (m + log2f(l)) * kLn2 : l == 0.f ? -INFINITY : l;
          if (partial)     // NaN as +inf: see the narrow kernel
            p.mid_lse[dst_q * p.hq + head] = l >= 0.f ? lse : INFINITY;
          else if (p.lse)
            p.lse[dst_q * p.hq + head] = lse;
        }
      } else {
        *abort_flag = 1;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
  }
}

template <typename T, typename CT, int D>
static int paged_wide_launch(const PagedParams& p, int max_wide, cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};
  auto kernel = paged_wide_kernel<T, CT, D>;
  const int rc = allow_smem(kernel, PwSmem<D>::BYTES, ready);
  if (rc != BE_OK) return rc;
  BE_CUDA_CHECK(launch_pdl(kernel, dim3((unsigned)max_wide * p.hkv), dim3(PW_THREADS),
                           PwSmem<D>::BYTES, st, p));
  return BE_OK;
}

}  // namespace be
