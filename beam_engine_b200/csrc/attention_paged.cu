// Paged attention for narrow tiles (up to 16 query-head rows) over 8-bit or 16-bit
// caches, with a causal limit, a sliding window and sinks; the plan is be_paged_plan's.
//
//   o_i = sum_t exp(x_it) v_t / sum_t exp(x_it),  x_it = sm_scale * q_i . k_t
//   over the tokens t that row i sees, in one pass with a running maximum.
//
// 8-bit caches hold codes: k_t = s_K c_t, v_t = s_V d_t with one scale per (page,
// KV head).  The codes become halves by one exact conversion per pair and the
// scales never touch them: s_K multiplies the score (it joins sm_scale), and s_V
// goes into the exponent, against a unit u = 2^lref that a warp's O is kept in,
//   sum_t exp(x_t) s_V,t d_t = u sum_t 2^(x'_t + a_t) d_t,  a = log2(s_V / u),  x' = x log2(e),
// and the denominator is the sum of those factors times 2^-a.  The factors are fp16 (steps of 2^-24 at
// least), so a must not take range from x': a stays in [0, 7], and the running maximum
// is taken 7 lower.  A token whose x' is the largest then has a factor of 1 or more whatever the
// scales of other pages are (which a value in another dim, or of a token that is not seen,
// may have set), and no factor passes 2^11.  Pages outside [u, 2^7 u] move u: O is
// multiplied by the old unit over the new one, an exact power of two in fp32.  Tokens of one step that
// no single u holds are taken in turns.  Scales may span 2^-40 to 2^40 (O stays below 2^127 when u
// falls that far: factors of 2^11 of codes of 2^9 over 2^18 tokens are 2^38).
// bf16 queries of an 8-bit cache are scaled per row by a power of two into half
// range (exact down to 2^-25 of the row's largest value: 8 significant bits above fp16's smallest
// step), so both products run in fp16 with fp32 sums; 16-bit caches use their own type.
//
// A warp takes 16 tokens at a time through a ring of its own in shared memory (cp.async by
// 16 bytes, no barrier between warps) into mma.sync fragments, tokens as the fragments' 16 rows and
// query rows as their 8 columns: S^T = K Q^T and O^T = V^T P^T, so that the few rows of a single
// token's heads fill half the products that the other way round needs (up to 8 rows; 16 take two
// blocks).  P^T turns from result to operand by a transpose of 8 x 8 halves.  The dims of a fragment
// may be in any order as long as Q and K (or V and O) agree, so a lane reads 16-byte pieces: lane
// (r, c) = (lane / 4, lane % 4) has pieces c, c + 4, ... of tokens r and r + 8 for S and piece r of
// tokens 2c, 2c + 1, 2c + 8, 2c + 9 for O; pieces are swizzled by the token so that both
// reads hit every bank once.  The ring keeps 2 or 3 steps in flight per warp (8 KB at 128 dims in
// 8 bits, 16 warps per SM); loading straight into registers kept one and ran at a quarter of
// HBM's rate (1 600 GB/s over 64 requests of up to 4 096 tokens).
//
// Bound: HBM for 16-bit caches.  64 requests, window 4096 + 4 of 16 000 tokens, bf16: 159 to 170 us, 6.3 to
// 6.75 TB/s; 64 requests of up to 4 096 tokens in 8 bits: 90 us, 4.5 TB/s (468 instructions for 16
// tokens' K and V, 64 of them conversions, for half the bytes; 412 and 86 us with log2 s_V whole in the
// exponent and no unit, which lost tokens).  Four warps of a CTA split the item's tokens and fold their states
// through shared memory; items that split a sequence leave partial rows for merge_kernel.
#include <atomic>

#include "common.cuh"

namespace be {

struct PagedParams {
  const int32_t* plan;   // header on the device
  const char* q;
  int64_t q_row_stride;
  const char* pool;
  const float* scale;    // [pages][2][hkv] of an 8-bit cache
  int num_pages, ps, hq, hkv, g;
  float scale_log2;
  char* out;
  int64_t out_row_stride;
  float* lse;
  float* mid_o;
  float* mid_lse;
  int out_vec16;         // out's rows are 16-byte aligned
  int merge_next;        // the merge is launched next: it may be prepared while these tiles run
};

struct E4M3 {};          // cache element tag
template <typename CT> struct CacheElt { static constexpr int bytes = 2; };
template <> struct CacheElt<E4M3> { static constexpr int bytes = 1; };

constexpr float kLazyMax = 8.f;       // factors up to 2^8 before O is rescaled
constexpr float kUnitSpan = 7.f;      // log2 of the V scales that one unit of O serves (8-bit caches)
constexpr float kLazyMax8 = 4.f;      // narrow tiles over 8 bits: factors up to 2^(7 + 4)
constexpr float kNoMax = -1e30f;      // running maximum of a row that has seen nothing

// Loads that stay where they are written: a plain load of constant memory is moved down to its
// first use, which puts its latency back into every step.
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0));
}
__device__ __forceinline__ int4 ld_early16(const void* p) {
  int4 v;
  asm volatile("ld.global.nc.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ int ld_early4(const int32_t* p) {
  int v;
  asm volatile("ld.global.nc.s32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float ld_early4(const float* p) {
  float v;
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float lg2(float x) {      // of normal numbers: the hardware's, exact for 2^n
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// An 8 x 8 block of halves, one row per four lanes, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  return __byte_perm(a, b, sel);
}
// true when one of the word's elements is not finite
template <typename CT>
__device__ __forceinline__ bool word_not_finite(uint32_t w) {
  if constexpr (std::is_same<CT, E4M3>::value) {
    const uint32_t m = w & 0x7f7f7f7fu;          // 0x7f: NaN (e4m3 has no infinities)
    return ((m + 0x01010101u) & 0x80808080u) != 0;
  } else if constexpr (std::is_same<CT, __half>::value) {
    return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
  } else {
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
  }
}

// Ring of one warp: stages of 16 K rows, 16 V rows, 16 + 16 scales and a word of valid tokens.
template <typename CT, int D, int NB>
struct PnRing {
  static constexpr int ROWB = D * CacheElt<CT>::bytes;
  static constexpr int STAGE = 2 * 16 * ROWB + 256;
  // up to 8 rows of 128 bytes: 4 CTAs per SM with 2 steps ahead beat 3 CTAs with 3 (shared prefixes with
  // 128 suffixes 38 us against 41; one sequence of 131 072 tokens 3 % slower)
  static constexpr int STAGES = ROWB <= 128 && NB == 2 ? 4 : 3;
  static constexpr int CTAS = ROWB > 128 ? 2 : NB == 1 ? 4 : 3;      // per SM
  static constexpr int FOLD = 4 * 8 * NB * (D + 4) * 4;   // the warps' O at the end
  static constexpr int BYTES = 4 * STAGES * STAGE > FOLD ? 4 * STAGES * STAGE : FOLD;
};

// T: type of q and out.  CT: E4M3 or T.  NB: blocks of 8 rows (1 or 2).
template <typename T, typename CT, int D, int NB>
__global__ void __launch_bounds__(128, PnRing<CT, D, NB>::CTAS) paged_narrow_kernel(const PagedParams p) {
  constexpr bool Q8 = std::is_same<CT, E4M3>::value;
  using MT = typename std::conditional<Q8, __half, T>::type;   // type of the products
  constexpr int EB = CacheElt<CT>::bytes;
  constexpr int ROWB = D * EB;                 // bytes of one (token, head) row
  constexpr int KP = ROWB / 64;                // 16-byte K pieces per lane and token
  constexpr int KW = 16 / EB;                  // dims per piece
  constexpr int VB = ROWB / 8 < 16 ? ROWB / 8 : 16;   // bytes per V piece
  constexpr int VP = ROWB / (8 * VB);          // V pieces per lane and token
  constexpr int VW = VB / EB;                  // dims per V piece
  constexpr int KS = D / 16;                   // k-steps of S = tiles of 16 dims of O
  constexpr int OLD = D + 4;
  using Ring = PnRing<CT, D, NB>;
  constexpr int CHR = ROWB / 16;               // 16-byte chunks per row
  extern __shared__ __align__(128) char ring_raw[];
  float (*sO)[8 * NB][OLD] = reinterpret_cast<float (*)[8 * NB][OLD]>(ring_raw);
  __shared__ float sM[4][8 * NB], sL[4][8 * NB], sU[4];

  pdl_wait();
  if (p.merge_next) pdl_trigger();   // the merge waits for this grid; another kernel might not
  const be_paged_plan_info* hdr = reinterpret_cast<const be_paged_plan_info*>(p.plan);
  const int n_wide = hdr->n_work_wide;
  const int item = blockIdx.x / p.hkv, kvh = blockIdx.x - item * p.hkv;
  if (item >= hdr->n_work - n_wide) return;
  const be_paged_item w =
      reinterpret_cast<const be_paged_item*>(p.plan + hdr->off_work)[n_wide + item];
  const int32_t* kvlist = p.plan + hdr->off_kvlist + w.kv_off;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
  const int g = p.g, rows = w.q_len * g;
  const bool causal = (w.flags & BE_ITEM_CAUSAL) != 0;
  const bool window = w.window >= 0;
  if (rows > 8 * NB) {                         // a plan made for higher tiles
    if (tid == 0) flag_range_error();
    return;
  }

  // ---- Q fragments (second operand): row 8 b + r, this lane's D / 4 dims as 16-bit pairs ----
  uint32_t qb[NB][D / 8];
  float up_r[NB];                              // 1 / (what the row's products are scaled by)
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int row = r + 8 * b;
    uint32_t (&raw)[D / 8] = qb[b];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) raw[i] = 0;
    if (row < rows) {
      const T* src = reinterpret_cast<const T*>(p.q) + (w.q_begin + row / g) * p.q_row_stride +
                     (int64_t)(kvh * g + row % g) * D;
#pragma unroll
      for (int k = 0; k < KP; ++k)
#pragma unroll
        for (int x = 0; x < KW / 8; ++x) {
          const int4 v = *reinterpret_cast<const int4*>(src + k * 4 * KW + c * KW + x * 8);
          const int o = k * (KW / 2) + x * 4;
          raw[o] = v.x; raw[o + 1] = v.y; raw[o + 2] = v.z; raw[o + 3] = v.w;
        }
    }
    up_r[b] = p.scale_log2;
    if constexpr (Q8 && std::is_same<T, __nv_bfloat16>::value) {
      float mx = 0.f;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[i]));
        mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // 2^(8 - floor(log2 mx)): the row's largest value lands in [2^8, 2^9)
      int e = (int)(__float_as_uint(mx) >> 23) - 127;
      e = mx < INFINITY ? min(max(e, -110), 110) : 0;
      const float up = __uint_as_float((uint32_t)(8 - e + 127) << 23);
      up_r[b] *= __uint_as_float((uint32_t)(e - 8 + 127) << 23);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[i]));
        const __half2 x = __floats2half2_rn(f.x * up, f.y * up);
        raw[i] = *reinterpret_cast<const uint32_t*>(&x);
      }
    }
  }
  // from here a lane's rows are 8 b + 2 c + e: columns of the score fragments
  float row_scale[NB][2];
  int pos_r[NB][2];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      row_scale[b][e] = __shfl_sync(0xffffffffu, up_r[b], (2 * c + e) * 4);
      pos_r[b][e] = w.pos0 + w.pos_step * ((8 * b + 2 * c + e) / g);
    }
  const int pos_hi = w.pos0 + w.pos_step * (w.q_len - 1);

  const int64_t row_step = (int64_t)p.hkv * ROWB;             // bytes between a page's tokens
  const char* base = p.pool + (int64_t)kvh * ROWB;
  char* ring = ring_raw + warp * (Ring::STAGES * Ring::STAGE);
  const int ps_shift = (p.ps & (p.ps - 1)) == 0 ? __ffs(p.ps) - 1 : -1;
  auto token_t = [&](int v) { return v + (v >= w.n0 ? w.shift : 0); };
  // place of token t's row in the ring (8-bit rows of 64 dims: two lie in one line of banks, so even
  // and odd tokens go to different halves) and of its chunk
  auto row_at = [](int t) { return (ROWB == 64 ? (t >> 1) | ((t & 1) << 3) : t) * ROWB; };
  auto chunk_at = [](int t, int ch) {
    return (ROWB == 64 ? ch ^ (((t >> 2) & 1) << 1) : ch ^ ((t & 6) ^ ((t & 1) << 2))) << 4;
  };
  auto page_of = [&](int v) -> int {           // page id of token v + (lane & 15), if it is there
    const int t = token_t(min(v + (lane & 15), w.v_end - 1));
    return ld_early4(kvlist + (ps_shift >= 0 ? t >> ps_shift : t / p.ps));
  };
  // this lane's part of a step's copies: chunk ch of tokens k0, k0 + KSTEP, ...
  constexpr int KSTEP = 32 / CHR, COPIES = 16 / KSTEP;
  const int k0 = lane / CHR, ch = lane % CHR;
  const uint32_t step_bytes = (uint32_t)row_step;
  const int64_t v_plane = row_step * p.ps;
  const char* src0 = base + ch * 16;
  // (the compiler does not see that the swizzle of a lane's tokens has few values)
  uint32_t copy_at[COPIES > 1 ? 2 : 1];
#pragma unroll
  for (int i = 0; i < (COPIES > 1 ? 2 : 1); ++i)
    copy_at[i] = smem_u32(ring) + row_at(k0 + i * KSTEP) + chunk_at(k0 + i * KSTEP, ch);
  constexpr bool TWO = ROWB == 128;            // tokens 2 KSTEP = 8 apart: the same swizzle
  // Requests the 16 tokens from v0 into stage st; tokens that are not there are zeros.
  auto issue = [&](int st, int v0, int page) {
    if (v0 < w.v_end) {
      char* dst = ring + st * Ring::STAGE;
      const int v = v0 + (lane & 15), t = token_t(v);
      const bool has = v < w.v_end && (unsigned)page < (unsigned)p.num_pages;
      const int row = has ? page * 2 * p.ps + (ps_shift >= 0 ? t & (p.ps - 1) : t % p.ps) : 0;
      const unsigned valid = __ballot_sync(0xffffffffu, has) & 0xffffu;
      if (valid != (w.v_end - v0 >= 16 ? 0xffffu : (1u << (w.v_end - v0)) - 1u)) flag_range_error();
      if (lane == 0) *reinterpret_cast<unsigned*>(dst + 2 * 16 * ROWB + 128) = valid;
#pragma unroll
      for (int i = 0; i < COPIES; ++i) {
        const int k = k0 + i * KSTEP;
        const uint32_t rk = __shfl_sync(0xffffffffu, (uint32_t)row, k);
        const char* src = src0 + (uint64_t)rk * step_bytes;
        const uint32_t to = TWO ? copy_at[i & 1] + st * Ring::STAGE + (i >> 1) * (2 * KSTEP * ROWB)
                                : smem_u32(dst + row_at(k) + chunk_at(k, ch));
        const bool there = (valid >> k) & 1;
        cp_async16(to, src, there);
        cp_async16(to + 16 * ROWB, src + v_plane, there);
      }
      if constexpr (Q8) {
        const float* s = p.scale + (has ? (int64_t)page * 2 * p.hkv + kvh + (lane < 16 ? 0 : p.hkv) : 0);
        cp_async4(smem_u32(dst + 2 * 16 * ROWB + lane * 4), s, has);
      }
    }
    cp_commit();
  };

  // O^T: tile j holds dims i = 2 j and 2 j + 1 of this lane's V pieces (the fragment's rows r and
  // r + 8), columns 8 b + 2c + {0, 1}
  float o[NB][KS][4];
  float m[NB][2], l[NB][2];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int j = 0; j < KS; ++j) o[b][j][0] = o[b][j][1] = o[b][j][2] = o[b][j][3] = 0.f;
    m[b][0] = m[b][1] = kNoMax;
    l[b][0] = l[b][1] = 0.f;
  }

  constexpr float kHead = Q8 ? kUnitSpan : 0.f, kLazy = Q8 ? kLazyMax8 : kLazyMax;
  float lref = -1000.f;                        // log2 of O's unit: the first step sets it
  int v0 = w.v_begin + warp * 16, st = 0;
  int page_next = page_of(v0);
#pragma unroll
  for (int j = 0; j < Ring::STAGES - 1; ++j) {
    const int page = page_next;
    page_next = page_of(v0 + 64 * (j + 1));
    issue(j, v0 + 64 * j, page);
  }
  const int k_at = row_at(r) + chunk_at(r, c);
#pragma unroll 1
  for (; v0 < w.v_end; v0 += 64) {
    cp_wait<Ring::STAGES - 2>();
    __syncwarp();
    // the stage read in the step before takes the tokens 3 (2) steps ahead
    const int page = page_next;
    page_next = page_of(v0 + 64 * Ring::STAGES);
    issue(st == 0 ? Ring::STAGES - 1 : st - 1, v0 + 64 * (Ring::STAGES - 1), page);
    const char* stage = ring + st * Ring::STAGE;
    unsigned turn = 0xffffu, later = 0;        // tokens of this pass over the step; of passes to come
    for (;;) {
      // ---- S^T = K Q^T: 16 tokens x 8 NB rows; s[b][i]: token r + 8 (i >> 1), row 8 b + 2c + (i & 1) ----
      float s[NB][4] = {};
#pragma unroll
      for (int k = 0; k < KP; ++k) {
        const int at = ROWB == 64 ? 0 : k_at ^ (k * 64);       // pieces 4 apart: one bit of the chunk
        const uint4 x0 = *reinterpret_cast<const uint4*>(
            stage + (ROWB == 64 ? row_at(r) + chunk_at(r, k * 4 + c) : at));
        const uint4 x1 = *reinterpret_cast<const uint4*>(
            stage + (ROWB == 64 ? row_at(r + 8) + chunk_at(r + 8, k * 4 + c) : at + 8 * ROWB));
        const uint32_t wa[4] = {x0.x, x0.y, x0.z, x0.w}, wb[4] = {x1.x, x1.y, x1.z, x1.w};
        if constexpr (Q8) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t a[4] = {e4m3x2_to_h2(wa[x] & 0xffffu), e4m3x2_to_h2(wb[x] & 0xffffu),
                                   e4m3x2_to_h2(wa[x] >> 16), e4m3x2_to_h2(wb[x] >> 16)};
#pragma unroll
            for (int b = 0; b < NB; ++b)
              mma16816<MT>(s[b], a, qb[b][2 * (k * 4 + x)], qb[b][2 * (k * 4 + x) + 1]);
          }
        } else {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t a[4] = {wa[2 * x], wb[2 * x], wa[2 * x + 1], wb[2 * x + 1]};
#pragma unroll
            for (int b = 0; b < NB; ++b)
              mma16816<MT>(s[b], a, qb[b][2 * (k * 2 + x)], qb[b][2 * (k * 2 + x) + 1]);
          }
        }
      }
      // ---- scores in base 2, masked ----
      const unsigned valid = *reinterpret_cast<const unsigned*>(stage + 2 * 16 * ROWB + 128) & turn;
      const int t_lo = token_t(v0), t_hi = token_t(v0 + 15);
      const bool full = valid == 0xffffu && (!causal || t_hi <= w.pos0) &&
                        (!window || t_lo >= pos_hi - w.window || t_hi < w.sink_end);
      float mult[2] = {1.f, 1.f}, add[2] = {0.f, 0.f}, rsv[2] = {1.f, 1.f};   // tokens r, r + 8
      bool grew = false;
      if constexpr (Q8) {
        const float* sc = reinterpret_cast<const float*>(stage + 2 * 16 * ROWB);
        // a V scale of 0 (a block never written) stands for values of 0: any scale will do
        mult[0] = sc[r];
        add[0] = lg2(fmaxf(sc[16 + r], 9.0949470177e-13f)) - lref;         // 2^-40
        rsv[0] = ex2(-add[0]);
        if (t_hi - t_lo == 15 && ((p.ps | t_lo) & 15) == 0) {              // one page
          mult[1] = mult[0];
          add[1] = add[0];
          rsv[1] = rsv[0];
        } else {
          mult[1] = sc[r + 8];
          add[1] = lg2(fmaxf(sc[24 + r], 9.0949470177e-13f)) - lref;
          rsv[1] = ex2(-add[1]);
        }
        grew = fabsf(add[0] - 0.5f * kUnitSpan) > 0.5f * kUnitSpan ||
               fabsf(add[1] - 0.5f * kUnitSpan) > 0.5f * kUnitSpan;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int h = i >> 1, e = i & 1;
          float x = Q8 ? fmaf(s[b][i], row_scale[b][e] * mult[h], add[h]) : s[b][i] * row_scale[b][e];
          if (!full) {
            const int k = r + 8 * h, t = token_t(v0 + k);
            const bool see = ((valid >> k) & 1) && (!causal || t <= pos_r[b][e]) &&
                             (!window || t >= pos_r[b][e] - w.window || t < w.sink_end);
            x = see ? x : -INFINITY;
          }
          s[b][i] = x;
          grew |= x > m[b][e] + (kHead + kLazy);
        }
      // ---- O's unit moves when a page's scale leaves its span, the running maximum only when a factor
      // would pass 2^8 (2^11) ----
      if (__any_sync(0xffffffffu, grew)) {
        if constexpr (Q8) {
          const bool has0 = (valid >> r) & 1, has1 = (valid >> (r + 8)) & 1;
          float lo = fminf(has0 ? add[0] : INFINITY, has1 ? add[1] : INFINITY);
          float hi = fmaxf(has0 ? add[0] : -INFINITY, has1 ? add[1] : -INFINITY);
#pragma unroll
          for (int off = 4; off < 32; off *= 2) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
          }
          if (lo <= hi && (lo < 0.f || hi > kUnitSpan)) {       // the same in every lane
            // the tokens' span in the middle of the new unit's; from the smallest if it is wider: the
            // tokens past it wait for a turn of their own
            const float from = floorf(lo), slack = kUnitSpan - (hi - from);
            const float by = slack >= 0.f ? from - floorf(0.5f * slack) : from;
            const float f = ex2(fminf(-by, 126.f));
            lref += by;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[b][j][i] *= f;
            // (lanes of one r agree: lane 4 r tells of tokens r and r + 8)
            unsigned out = __ballot_sync(0xffffffffu, c == 0 && has0 && add[0] - by > kUnitSpan) |
                           __ballot_sync(0xffffffffu, c == 1 && has1 && add[1] - by > kUnitSpan);
            unsigned wait = 0;
            for (int k = 0; k < 8; ++k)
              wait |= ((out >> (4 * k)) & 1) << k | ((out >> (4 * k + 1)) & 1) << (k + 8);
            later |= wait;
            turn = valid & ~wait;
            continue;                                           // the scores again, in the new unit
          }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(s[b][e], s[b][2 + e]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mx = fmaxf(mx - kHead, m[b][e]);
            const float f = ex2(m[b][e] - mx);
            m[b][e] = mx;
            l[b][e] *= f;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
              o[b][j][e] *= f;
              o[b][j][2 + e] *= f;
            }
          }
      }
      // P^T as the second operand: the fragment's 8 x 8 blocks of halves, transposed
      uint32_t pb[NB][2];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float a0 = ex2(s[b][2 * h] - m[b][0]), a1 = ex2(s[b][2 * h + 1] - m[b][1]);
          l[b][0] = fmaf(a0, rsv[h], l[b][0]);
          l[b][1] = fmaf(a1, rsv[h], l[b][1]);
          s[b][2 * h] = a0;
          s[b][2 * h + 1] = a1;
          pb[b][h] = transpose8(pack2<MT>(a0, a1));
        }
      // ---- V fragments' words: tokens 2c, 2c + 1, 2c + 8, 2c + 9 ----
      uint32_t vraw[4][VP * VB / 4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int t = (n >> 1) * 8 + 2 * c + (n & 1);
        const char* src = stage + 16 * ROWB + row_at(t);
#pragma unroll
        for (int k = 0; k < VP; ++k) {
          if constexpr (VB == 16) {
            const uint4 x = *reinterpret_cast<const uint4*>(src + chunk_at(t, k * 8 + r));
            vraw[n][4 * k] = x.x; vraw[n][4 * k + 1] = x.y;
            vraw[n][4 * k + 2] = x.z; vraw[n][4 * k + 3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(src + chunk_at(t, r >> 1) + (r & 1) * 8);
            vraw[n][0] = x.x; vraw[n][1] = x.y;
          }
        }
      }
      // ---- values that are not finite and not seen by every row: out of the product (0 * NaN is
      // NaN), added to the rows that see them ----
      if (!full) {
        bool odd = false;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int k = 0; k < VP * VB / 4; ++k) odd |= word_not_finite<CT>(vraw[n][k]);
        if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            bool mine = false;
#pragma unroll
            for (int k = 0; k < VP * VB / 4; ++k) mine |= word_not_finite<CT>(vraw[n][k]);
            // the token's row is spread over the lanes with this c
            unsigned any = __ballot_sync(0xffffffffu, mine);
            any &= 0x11111111u << c;
            if (any)
#pragma unroll
              for (int k = 0; k < VP * VB / 4; ++k) vraw[n][k] = 0;
          }
#pragma unroll 1
          for (int k = 0; k < 16; ++k) {
            if (!((valid >> k) & 1)) continue;
            const char* row_v = stage + 16 * ROWB + row_at(k);
            bool has = false;
            for (int b = lane * 4; b < ROWB; b += 128)
              has |= word_not_finite<CT>(*reinterpret_cast<const uint32_t*>(row_v + b));
            if (!__any_sync(0xffffffffu, has)) continue;
            const int src = (k & 7) * 4 + c;     // the lane with this token's probabilities
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              const float a0 = __shfl_sync(0xffffffffu, s[b][0], src), a1 = __shfl_sync(0xffffffffu, s[b][1], src);
              const float a2 = __shfl_sync(0xffffffffu, s[b][2], src), a3 = __shfl_sync(0xffffffffu, s[b][3], src);
              const float q0 = k < 8 ? a0 : a2, q1 = k < 8 ? a1 : a3;
#pragma unroll
              for (int i = 0; i < 2 * KS; ++i) {
                const int at = ((i / VW) * 8 * VW + r * VW + i % VW) * EB;    // byte of the row
                const char* src_v = row_v + chunk_at(k, at >> 4) + (at & 15);
                float val;
                if constexpr (Q8) {
                  const uint32_t h2 = e4m3x2_to_h2(*reinterpret_cast<const uint8_t*>(src_v));
                  val = __low2float(*reinterpret_cast<const __half2*>(&h2));
                } else {
                  val = to_f(*reinterpret_cast<const T*>(src_v));
                }
                float* acc = &o[b][i / 2][(i & 1) * 2];
                if (q0 > 0.f) acc[0] = fmaf(q0, val, acc[0]);
                if (q1 > 0.f) acc[1] = fmaf(q1, val, acc[1]);
              }
            }
          }
        }
      }
      // ---- O^T += V^T P^T ----
#pragma unroll
      for (int k = 0; k < VP * VB / 4; ++k) {
        if constexpr (Q8) {
          const uint32_t a01 = prmt(vraw[0][k], vraw[1][k], 0x5140), a23 = prmt(vraw[0][k], vraw[1][k], 0x7362);
          const uint32_t b01 = prmt(vraw[2][k], vraw[3][k], 0x5140), b23 = prmt(vraw[2][k], vraw[3][k], 0x7362);
          const uint32_t x[4] = {e4m3x2_to_h2(a01 & 0xffffu), e4m3x2_to_h2(a01 >> 16),
                                 e4m3x2_to_h2(b01 & 0xffffu), e4m3x2_to_h2(b01 >> 16)};
          const uint32_t y[4] = {e4m3x2_to_h2(a23 & 0xffffu), e4m3x2_to_h2(a23 >> 16),
                                 e4m3x2_to_h2(b23 & 0xffffu), e4m3x2_to_h2(b23 >> 16)};
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            mma16816<MT>(o[b][2 * k], x, pb[b][0], pb[b][1]);
            mma16816<MT>(o[b][2 * k + 1], y, pb[b][0], pb[b][1]);
          }
        } else {
          const uint32_t x[4] = {prmt(vraw[0][k], vraw[1][k], 0x5410), prmt(vraw[0][k], vraw[1][k], 0x7632),
                                 prmt(vraw[2][k], vraw[3][k], 0x5410), prmt(vraw[2][k], vraw[3][k], 0x7632)};
#pragma unroll
          for (int b = 0; b < NB; ++b) mma16816<MT>(o[b][k], x, pb[b][0], pb[b][1]);
        }
      }
      if (!Q8 || later == 0) break;
      turn = later;
      later = 0;
    }
    st = st + 1 == Ring::STAGES ? 0 : st + 1;
  }
  cp_wait<0>();
  __syncthreads();                             // every ring is read: O goes there

  // ---- fold the four warps ----
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int off = 4; off < 32; off *= 2) l[b][e] += __shfl_xor_sync(0xffffffffu, l[b][e], off);
      if (lane == 0 && b == 0 && e == 0) sU[warp] = Q8 ? ex2(lref) : 1.f;
      if (r == 0) {
        sM[warp][8 * b + 2 * c + e] = m[b][e];
        sL[warp][8 * b + 2 * c + e] = l[b][e];
      }
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i)
        sO[warp][8 * b + 2 * c + e][(i / VW) * 8 * VW + r * VW + i % VW] = o[b][i / 2][(i & 1) * 2 + e];
    }
  __syncthreads();
  constexpr int TPR = 128 / (8 * NB);          // threads per row
  const int row = tid / TPR, d0 = (tid % TPR) * 4;
  if (row >= rows) return;
  const float mx = fmaxf(fmaxf(sM[0][row], sM[1][row]), fmaxf(sM[2][row], sM[3][row]));
  float f[4], den = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[k] = ex2(sM[k][row] - mx);
    den += f[k] * sL[k][row];
    if constexpr (Q8) f[k] *= sU[k];
  }
  const float inv = den != 0.f ? 1.f / den : 0.f;
  const int qi = row / g, head = kvh * g + row % g;
  const int64_t dst_q = w.part_base < 0 ? w.q_begin + qi : w.part_base + qi;
#pragma unroll
  for (int d = d0; d < D; d += 4 * TPR) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 x = *reinterpret_cast<const float4*>(&sO[k][row][d]);
      acc.x += f[k] * x.x; acc.y += f[k] * x.y; acc.z += f[k] * x.z; acc.w += f[k] * x.w;
    }
    acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
    if (w.part_base < 0)
      *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + dst_q * p.out_row_stride +
                                (int64_t)head * D + d) =
          make_uint2(pack2<T>(acc.x, acc.y), pack2<T>(acc.z, acc.w));
    else
      *reinterpret_cast<float4*>(p.mid_o + (dst_q * p.hq + head) * D + d) = acc;
  }
  if (tid % TPR == 0) {
    const float lse = den > 0.f ? (mx + log2f(den)) * kLn2 : den == 0.f ? -INFINITY : den;
    // a NaN partial row is merged as +inf: the merge takes the maximum over its parts, which
    // passes over NaN, and inf - inf makes the row NaN there
    if (w.part_base >= 0)
      p.mid_lse[dst_q * p.hq + head] = den >= 0.f ? lse : INFINITY;
    else if (p.lse)
      p.lse[dst_q * p.hq + head] = lse;
  }
}

// merge_kernel's work with a CTA per (query, head): four warps take every fourth partial row.
// A long sequence split over the GPU leaves dozens of parts for a few rows, and one warp
// walking them is latency alone (one sequence of 131 072 tokens, 8-bit, when this came: 66 us with it, 59 with this).
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_merge_kernel(const PagedParams p) {
  __shared__ __align__(16) float sO[4][D];
  __shared__ float sM[4], sL[4];
  pdl_wait();
  const be_paged_plan_info* hdr = reinterpret_cast<const be_paged_plan_info*>(p.plan);
  const int b = blockIdx.x / p.hq, head = blockIdx.x - b * p.hq;
  if (b >= hdr->n_merge) return;
  const int qi = p.plan[hdr->off_merge_q + b];
  const int p0 = p.plan[hdr->off_merge_ptr + b], p1 = p.plan[hdr->off_merge_ptr + b + 1];
  const int32_t* parts = p.plan + hdr->off_merge_parts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int DL = D / 32;                   // floats per lane
  float acc[DL] = {}, m = -INFINITY, l = 0.f;
  for (int k0 = p0 + warp; k0 < p1; k0 += 16) {   // 4 parts of this warp at once
    float e[4], x[4][DL];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = k0 + 4 * u;
      const int64_t row = k < p1 ? (int64_t)parts[k] * p.hq + head : -1;
      e[u] = row >= 0 ? p.mid_lse[row] : -INFINITY;
#pragma unroll
      for (int d = 0; d < DL; ++d) x[u][d] = row >= 0 ? p.mid_o[row * D + lane * DL + d] : 0.f;
    }
    float to = m;
#pragma unroll
    for (int u = 0; u < 4; ++u) to = fmaxf(to, e[u]);
    if (to == -INFINITY) continue;
    const float f = m == -INFINITY ? 0.f : expf(m - to);
    m = to;
    l *= f;
#pragma unroll
    for (int d = 0; d < DL; ++d) acc[d] *= f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (e[u] == -INFINITY) continue;         // empty: its row counts for nothing, whatever it holds
      const float g = expf(e[u] - to);
      l += g;
#pragma unroll
      for (int d = 0; d < DL; ++d) acc[d] = fmaf(g, x[u][d], acc[d]);
    }
  }
#pragma unroll
  for (int d = 0; d < DL; ++d) sO[warp][lane * DL + d] = acc[d];
  if (lane == 0) {
    sM[warp] = m;
    sL[warp] = l;
  }
  __syncthreads();
  const float mx = fmaxf(fmaxf(sM[0], sM[1]), fmaxf(sM[2], sM[3]));
  float f[4], den = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[k] = sM[k] == -INFINITY ? 0.f : expf(sM[k] - mx);
    den += f[k] * sL[k];
  }
  for (int d = threadIdx.x; d < D; d += 128) {
    const float o = f[0] * sO[0][d] + f[1] * sO[1][d] + f[2] * sO[2][d] + f[3] * sO[3][d];
    reinterpret_cast<T*>(p.out)[qi * p.out_row_stride + (int64_t)head * D + d] =
        from_f<T>(den != 0.f ? o / den : 0.f);
  }
  if (p.lse && threadIdx.x == 0)
    p.lse[(int64_t)qi * p.hq + head] = den == 0.f ? -INFINITY : mx + logf(den);
}

// Raises a kernel's shared-memory limit, once per device.
template <typename K>
static int allow_smem(K kernel, int bytes, std::atomic<uint64_t>& ready) {
  int dev = 0;
  BE_CUDA_CHECK(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load() & bit)) {
    BE_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    ready.fetch_or(bit);
  }
  return BE_OK;
}

template <typename T, typename CT, int D, int NB>
static int paged_narrow_launch(const PagedParams& p, dim3 grid, cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};
  constexpr int bytes = PnRing<CT, D, NB>::BYTES;
  const int rc = allow_smem(paged_narrow_kernel<T, CT, D, NB>, bytes, ready);
  if (rc != BE_OK) return rc;
  BE_CUDA_CHECK(launch_pdl(paged_narrow_kernel<T, CT, D, NB>, grid, dim3(128), bytes, st, p));
  return BE_OK;
}

template <typename T, typename CT, int D>
static int paged_wide_launch(const PagedParams& p, int max_wide, cudaStream_t st);

template <typename T>
static int paged_launch(const PagedParams& p, bool q8, int D, int max_wide, int max_narrow,
                        int rows, int max_merge, cudaStream_t st) {
  if (max_wide > 0) {
    int rc;
    if (q8)
      rc = D == 128 ? paged_wide_launch<T, E4M3, 128>(p, max_wide, st)
                    : paged_wide_launch<T, E4M3, 64>(p, max_wide, st);
    else
      rc = D == 128 ? paged_wide_launch<T, T, 128>(p, max_wide, st)
                    : paged_wide_launch<T, T, 64>(p, max_wide, st);
    if (rc != BE_OK) return rc;
  }
  if (max_narrow > 0) {
    const dim3 grid((unsigned)max_narrow * p.hkv);   // heads of an item next to each other
    auto go = [&](auto elt, auto dim) {
      using CT = decltype(elt);
      constexpr int DD = decltype(dim)::value;
      return rows <= 8 ? paged_narrow_launch<T, CT, DD, 1>(p, grid, st)
                       : paged_narrow_launch<T, CT, DD, 2>(p, grid, st);
    };
    using D128 = std::integral_constant<int, 128>;
    using D64 = std::integral_constant<int, 64>;
    const int rc = q8 ? (D == 128 ? go(E4M3{}, D128{}) : go(E4M3{}, D64{}))
                      : (D == 128 ? go(T{}, D128{}) : go(T{}, D64{}));
    if (rc != BE_OK) return rc;
  }
  // a CTA per row while that is a few waves of CTAs, a warp per row for prompts' many rows
  if (max_merge > 0 && (int64_t)max_merge * p.hq <= 148 * 32) {
    if (D == 128)
      BE_CUDA_CHECK(launch_pdl(paged_merge_kernel<T, 128>, dim3(max_merge * p.hq), dim3(128), 0, st, p));
    else
      BE_CUDA_CHECK(launch_pdl(paged_merge_kernel<T, 64>, dim3(max_merge * p.hq), dim3(128), 0, st, p));
  } else if (max_merge > 0) {
    const int items = max_merge * p.hq;
    BE_CUDA_CHECK(launch_pdl(merge_kernel<T>, dim3((items + 3) / 4), dim3(128), 0, st,
                             (const int32_t*)nullptr, (const int32_t*)nullptr,
                             (const int32_t*)nullptr, max_merge, (const float*)p.mid_o,
                             (const float*)p.mid_lse, p.hq, D, p.out, p.out_row_stride, p.lse,
                             p.plan));
  }
  return BE_OK;
}

}  // namespace be

using namespace be;

extern "C" int be_paged_attn_run(const be_paged_attn_args* args) {
  if (!args) {
    set_error("be_paged_attn_run: null pointer");
    return BE_EINVAL;
  }
  const be_paged_attn_args& a = *args;
  const int max_wide = a.max_wide, max_narrow = a.max_narrow, max_merge = a.max_merge;
  const int page_size = a.page_size, num_pages = a.num_pages, head_dim = a.head_dim;
  const int num_qo_heads = a.num_qo_heads, num_kv_heads = a.num_kv_heads, dtype = a.dtype;
  if (max_wide < 0 || max_narrow < 0 || a.narrow_rows < 0 || a.narrow_rows > 16 || max_merge < 0 ||
      a.max_parts < 0 || page_size < 1 || num_pages < 1 || num_kv_heads < 1 || num_kv_heads > 1024 || num_qo_heads < 1 ||
      std::max(max_wide, max_narrow) > (1 << 20) ||
      num_qo_heads % num_kv_heads) {
    set_error("be_paged_attn_run: invalid shape");
    return BE_EINVAL;
  }
  // kernels number a pool's token rows in 31 bits, its (token, head) rows in 32
  const int64_t token_rows = (int64_t)num_pages * 2 * std::min(page_size, 1 << 24);
  if (token_rows > INT32_MAX || token_rows * num_kv_heads >= UINT32_MAX) {
    set_error("be_paged_attn_run: a pool of %d pages of %d tokens is too large", num_pages, page_size);
    return BE_EINVAL;
  }
  if ((dtype != BE_BF16 && dtype != BE_F16) || (a.cache_dtype != BE_E4M3 && a.cache_dtype != dtype)) {
    set_error("be_paged_attn_run: queries are bf16 or fp16, the cache e4m3 or of their type");
    return BE_EINVAL;
  }
  if (head_dim != 64 && head_dim != 128) {
    set_error("be_paged_attn_run: head_dim %d is not 64 or 128", head_dim);
    return BE_EINVAL;
  }
  if (num_qo_heads / num_kv_heads > 128) {
    set_error("be_paged_attn_run: %d query heads per KV head (at most 128)",
              num_qo_heads / num_kv_heads);
    return BE_EINVAL;
  }
  if (max_wide + max_narrow + max_merge == 0) return BE_OK;
  if (!a.plan_dev || !a.q || !a.paged_kv_cache || !a.out || (a.max_parts > 0 && (!a.mid_o || !a.mid_lse)) ||
      (a.cache_dtype == BE_E4M3) != (a.kv_scale != nullptr)) {
    set_error("be_paged_attn_run: null pointer (an 8-bit cache needs kv_scale, another has none)");
    return BE_EINVAL;
  }
  if (((uintptr_t)a.q | (uintptr_t)a.paged_kv_cache | (uintptr_t)a.mid_o) % 16 || (uintptr_t)a.out % 8 ||
      a.q_row_stride % 8 || a.out_row_stride % 4) {
    set_error("be_paged_attn_run: q and the cache must be 16-byte aligned, out 8-byte");
    return BE_EINVAL;
  }
  PagedParams p;
  p.plan = a.plan_dev;
  p.q = (const char*)a.q;
  p.q_row_stride = a.q_row_stride;
  p.pool = (const char*)a.paged_kv_cache;
  p.scale = a.kv_scale;
  p.num_pages = num_pages;
  p.ps = page_size;
  p.hq = num_qo_heads;
  p.hkv = num_kv_heads;
  p.g = num_qo_heads / num_kv_heads;
  p.scale_log2 = a.sm_scale * kLog2e;
  p.out = (char*)a.out;
  p.out_row_stride = a.out_row_stride;
  p.lse = a.lse;
  p.mid_o = a.mid_o;
  p.mid_lse = a.mid_lse;
  p.merge_next = max_merge > 0;
  p.out_vec16 = (uintptr_t)a.out % 16 == 0 && a.out_row_stride % 8 == 0;
  const bool q8 = a.cache_dtype == BE_E4M3;
  return dtype == BE_BF16
             ? paged_launch<__nv_bfloat16>(p, q8, head_dim, max_wide, max_narrow,
                                           a.narrow_rows, max_merge, (cudaStream_t)a.stream)
             : paged_launch<__half>(p, q8, head_dim, max_wide, max_narrow,
                                           a.narrow_rows, max_merge, (cudaStream_t)a.stream);
}
