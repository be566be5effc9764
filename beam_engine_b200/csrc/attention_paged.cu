// Paged attention for narrow tiles (up to 16 query-head rows) over 8-bit or 16-bit
// caches, with a causal limit, a sliding window and sinks; the plan is be_paged_plan's.
//
//   o_i = sum_t exp(x_it) v_t / sum_t exp(x_it),  x_it = sm_scale * q_i . k_t
//   over the tokens t that row i sees, in one pass with a running maximum.
//
// 8-bit caches hold codes: k_t = s_K c_t, v_t = s_V d_t with one scale per (page,
// KV head).  The codes become halves by one exact conversion per pair and the
// scales never touch them: s_K multiplies the score (it joins sm_scale), and s_V
// goes into the exponent,
//   sum_t exp(x_t) s_V,t d_t = sum_t 2^(x'_t + log2 s_V,t) d_t,  x' = x log2(e),
// so the running maximum is over x' + log2 s_V, every factor of the second product
// is at most 2^8, and the denominator is the sum of those factors divided by s_V.
// bf16 queries of an 8-bit cache are scaled per row by a power of two into half
// range (exact down to 2^-33 of the row's largest value), so both products run in
// fp16 with fp32 sums; 16-bit caches use their own type.
//
// A warp takes 16 tokens at a time straight from global memory into mma.sync
// fragments; nothing passes through shared memory before the end.  The dims of a
// fragment may be in any order as long as Q and K (or V and O) agree, so each lane
// loads 16-byte pieces: lane (r, c) = (lane / 4, lane % 4) holds token r's pieces c, c + 4, ...
// for S = Q K^T and piece r of tokens 2c, 2c + 1, 2c + 8, 2c + 9 for O = P V; whole
// rows of a token and head are read by neighbouring lanes.  The next 16 tokens' K is
// requested once this step's S is done, the next V once its O is done.
//
// Bound: HBM.  Four warps of a CTA split the item's tokens and fold their states
// through shared memory; items that split a sequence leave partial rows for merge_kernel.
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
};

struct E4M3 {};          // cache element tag
template <typename CT> struct CacheElt { static constexpr int bytes = 2; };
template <> struct CacheElt<E4M3> { static constexpr int bytes = 1; };

constexpr float kLazyMax = 8.f;       // factors up to 2^8 before O is rescaled
constexpr float kNoMax = -1e30f;      // running maximum of a row that has seen nothing

// Loads that stay where they are written: a plain load of constant memory is moved down to its
// first use, which puts its latency back into every step.
__device__ __forceinline__ int4 ld_early16(const void* p) {
  int4 v;
  asm volatile("ld.global.nc.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_early8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
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

// T: type of q and out.  CT: E4M3 or T.
template <typename T, typename CT, int D>
__global__ void __launch_bounds__(128) paged_narrow_kernel(const PagedParams p) {
  constexpr bool Q8 = std::is_same<CT, E4M3>::value;
  using MT = typename std::conditional<Q8, __half, T>::type;   // type of the products
  constexpr int EB = CacheElt<CT>::bytes;
  constexpr int ROWB = D * EB;                 // bytes of one (token, head) row
  constexpr int KP = ROWB / 64;                // 16-byte K pieces per lane and token
  constexpr int KW = 16 / EB;                  // dims per piece
  constexpr int VB = ROWB / 8 < 16 ? ROWB / 8 : 16;   // bytes per V piece
  constexpr int VP = ROWB / (8 * VB);          // V pieces per lane and token
  constexpr int VW = VB / EB;                  // dims per V piece
  constexpr int KS = D / 16, NT = D / 8;       // k-steps of S, column tiles of O
  constexpr int OLD = D + 4;
  __shared__ __align__(16) float sO[4][16][OLD];
  __shared__ float sM[4][16], sL[4][16];

  pdl_wait();
  const be_attn_plan_info* hdr = reinterpret_cast<const be_attn_plan_info*>(p.plan);
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

  // ---- Q fragments: rows r and r + 8 ----
  uint32_t qa[KS][4];
  float row_scale[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = r + 8 * h;
    uint32_t raw[D / 8];                       // this lane's D / 4 dims, 16-bit pairs
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
    row_scale[h] = p.scale_log2;
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
      row_scale[h] *= __uint_as_float((uint32_t)(e - 8 + 127) << 23);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[i]));
        const __half2 x = __floats2half2_rn(f.x * up, f.y * up);
        raw[i] = *reinterpret_cast<const uint32_t*>(&x);
      }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qa[s][h] = raw[2 * s];
      qa[s][2 + h] = raw[2 * s + 1];
    }
  }

  const int64_t row_step = (int64_t)p.hkv * ROWB;             // bytes between a page's tokens
  const int64_t plane_step = row_step * p.ps;
  const char* base = p.pool + (int64_t)kvh * ROWB;

  // Token (lane & 15) of the step that starts at v0: its K row's byte offset (V is a
  // plane further), or -1 past the range and for a page that does not exist.
  auto locate = [&](int v0, float& sk, float& sv) -> int64_t {
    const int v = v0 + (lane & 15);
    sk = 0.f;
    sv = 0.f;
    if (v >= w.v_end) return -1;
    const int t = v + (v >= w.n0 ? w.shift : 0);
    const int pi = t / p.ps;
    const int page = kvlist[pi];
    if (page < 0 || page >= p.num_pages) {
      flag_range_error();
      return -1;
    }
    if constexpr (Q8) {
      const float* s = p.scale + (int64_t)page * 2 * p.hkv + kvh;
      sk = s[0];
      sv = s[p.hkv];
    }
    return (int64_t)page * 2 * plane_step + (int64_t)(t - pi * p.ps) * row_step;
  };

  int4 kraw[2][KP];
  uint32_t vraw[4][VP * VB / 4];
  auto load_k = [&](int64_t at) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int64_t o = __shfl_sync(0xffffffffu, at, n * 8 + r);
#pragma unroll
      for (int k = 0; k < KP; ++k)
        kraw[n][k] = o >= 0 ? ld_early16(base + o + k * 64 + c * 16) : make_int4(0, 0, 0, 0);
    }
  };
  auto load_v = [&](int64_t at) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int64_t o = __shfl_sync(0xffffffffu, at, (n >> 1) * 8 + 2 * c + (n & 1));
      const char* src = base + o + plane_step;
#pragma unroll
      for (int k = 0; k < VP; ++k) {
        if constexpr (VB == 16) {
          const int4 x = o >= 0 ? ld_early16(src + k * 128 + r * 16) : make_int4(0, 0, 0, 0);
          vraw[n][4 * k] = x.x; vraw[n][4 * k + 1] = x.y;
          vraw[n][4 * k + 2] = x.z; vraw[n][4 * k + 3] = x.w;
        } else {
          const uint2 x = o >= 0 ? ld_early8(src + r * 8) : make_uint2(0, 0);
          vraw[n][0] = x.x; vraw[n][1] = x.y;
        }
      }
    }
  };

  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {kNoMax, kNoMax}, l[2] = {0.f, 0.f};
  const int pos_r[2] = {w.pos0 + w.pos_step * (r / g), w.pos0 + w.pos_step * ((r + 8) / g)};
  const int pos_hi = w.pos0 + w.pos_step * (w.q_len - 1);

  int v0 = w.v_begin + warp * 16;
  float sk = 0.f, sv = 0.f;
  int64_t at = locate(v0, sk, sv);
  if (v0 < w.v_end) {
    load_k(at);
    load_v(at);
  }
  for (; v0 < w.v_end; v0 += 64) {
    float sk_next, sv_next;
    const int64_t at_next = locate(v0 + 64, sk_next, sv_next);
    // ---- S = Q K^T over 2 x 8 tokens ----
    float s[2][4] = {};
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int k = 0; k < KP; ++k) {
        const uint32_t wd[4] = {(uint32_t)kraw[n][k].x, (uint32_t)kraw[n][k].y,
                                (uint32_t)kraw[n][k].z, (uint32_t)kraw[n][k].w};
        if constexpr (Q8) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            mma16816<MT>(s[n], qa[k * 4 + x], e4m3x2_to_h2(wd[x] & 0xffffu),
                         e4m3x2_to_h2(wd[x] >> 16));
        } else {
          mma16816<MT>(s[n], qa[k * 2], wd[0], wd[1]);
          mma16816<MT>(s[n], qa[k * 2 + 1], wd[2], wd[3]);
        }
      }
    }
    load_k(at_next);
    // ---- scores in base 2, masked; x[n][i]: token n * 8 + 2c + (i & 1), row r + 8 (i >> 1) ----
    const unsigned valid = __ballot_sync(0xffffffffu, at >= 0);
    const int t_lo = v0 + (v0 >= w.n0 ? w.shift : 0);
    const int t_hi = v0 + 15 + (v0 + 15 >= w.n0 ? w.shift : 0);
    const bool full = (valid & 0xffffu) == 0xffffu && (!causal || t_hi <= w.pos0) &&
                      (!window || t_lo >= pos_hi - w.window || t_hi < w.sink_end);
    float rsv[2][2] = {{1.f, 1.f}, {1.f, 1.f}};
    float mult[2][2] = {{1.f, 1.f}, {1.f, 1.f}}, add[2][2] = {};
    if constexpr (Q8) {
      // a V scale of 0 (a block never written) stands for values of 0: any scale will do
      const float svc = fmaxf(sv, 9.0949470177e-13f);            // 2^-40
      const float lsv = log2f(svc), inv = 1.f / svc;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int src = n * 8 + 2 * c + e;
          mult[n][e] = __shfl_sync(0xffffffffu, sk, src);
          add[n][e] = __shfl_sync(0xffffffffu, lsv, src);
          rsv[n][e] = __shfl_sync(0xffffffffu, inv, src);
        }
    }
    bool grew = false;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int h = i >> 1, e = i & 1;
        float x = Q8 ? fmaf(s[n][i], row_scale[h] * mult[n][e], add[n][e]) : s[n][i] * row_scale[h];
        if (!full) {
          const int k = n * 8 + 2 * c + e, v = v0 + k;
          const int t = v + (v >= w.n0 ? w.shift : 0);
          const bool see = ((valid >> k) & 1) && (!causal || t <= pos_r[h]) &&
                           (!window || t >= pos_r[h] - w.window || t < w.sink_end);
          x = see ? x : -INFINITY;
        }
        s[n][i] = x;
        grew |= x > m[h] + kLazyMax;
      }
    // ---- the running maximum moves only when a factor would pass 2^8 ----
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mx = fmaxf(mx, m[h]);
        const float f = ex2(m[h] - mx);
        m[h] = mx;
        l[h] *= f;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          o[i][2 * h] *= f;
          o[i][2 * h + 1] *= f;
        }
      }
    }
    float pf[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pf[n][i] = ex2(s[n][i] - m[i >> 1]);
        l[i >> 1] = fmaf(pf[n][i], rsv[n][i & 1], l[i >> 1]);
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
        for (int k = 0; k < 16; ++k) {
          const int64_t off = __shfl_sync(0xffffffffu, at, k);
          if (off < 0) continue;
          const int src = (lane & 28) + ((k & 7) >> 1);
          const float q00 = __shfl_sync(0xffffffffu, pf[0][0], src), q01 = __shfl_sync(0xffffffffu, pf[0][1], src);
          const float q02 = __shfl_sync(0xffffffffu, pf[0][2], src), q03 = __shfl_sync(0xffffffffu, pf[0][3], src);
          const float q10 = __shfl_sync(0xffffffffu, pf[1][0], src), q11 = __shfl_sync(0xffffffffu, pf[1][1], src);
          const float q12 = __shfl_sync(0xffffffffu, pf[1][2], src), q13 = __shfl_sync(0xffffffffu, pf[1][3], src);
          const float p0 = k < 8 ? ((k & 1) ? q01 : q00) : ((k & 1) ? q11 : q10);
          const float p1 = k < 8 ? ((k & 1) ? q03 : q02) : ((k & 1) ? q13 : q12);
          const char* src_v = base + off + plane_step;
          bool has = false;
          for (int b = lane * 4; b < ROWB; b += 128)
            has |= word_not_finite<CT>(*reinterpret_cast<const uint32_t*>(src_v + b));
          if (!__any_sync(0xffffffffu, has)) continue;
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int d = (i / VW) * 8 * VW + (2 * c + e) * VW + i % VW;
              float val;
              if constexpr (Q8) {
                const uint32_t h2 = e4m3x2_to_h2(*reinterpret_cast<const uint8_t*>(src_v + d));
                val = __low2float(*reinterpret_cast<const __half2*>(&h2));
              } else {
                val = to_f(reinterpret_cast<const T*>(src_v)[d]);
              }
              if (p0 > 0.f) o[i][e] = fmaf(p0, val, o[i][e]);
              if (p1 > 0.f) o[i][2 + e] = fmaf(p1, val, o[i][2 + e]);
            }
        }
      }
    }
    // ---- O += P V ----
    uint32_t pa[4];
    pa[0] = pack2<MT>(pf[0][0], pf[0][1]);
    pa[1] = pack2<MT>(pf[0][2], pf[0][3]);
    pa[2] = pack2<MT>(pf[1][0], pf[1][1]);
    pa[3] = pack2<MT>(pf[1][2], pf[1][3]);
#pragma unroll
    for (int k = 0; k < VP * VB / 4; ++k) {
      if constexpr (Q8) {
        const uint32_t a01 = prmt(vraw[0][k], vraw[1][k], 0x5140), a23 = prmt(vraw[0][k], vraw[1][k], 0x7362);
        const uint32_t b01 = prmt(vraw[2][k], vraw[3][k], 0x5140), b23 = prmt(vraw[2][k], vraw[3][k], 0x7362);
        mma16816<MT>(o[4 * k], pa, e4m3x2_to_h2(a01 & 0xffffu), e4m3x2_to_h2(b01 & 0xffffu));
        mma16816<MT>(o[4 * k + 1], pa, e4m3x2_to_h2(a01 >> 16), e4m3x2_to_h2(b01 >> 16));
        mma16816<MT>(o[4 * k + 2], pa, e4m3x2_to_h2(a23 & 0xffffu), e4m3x2_to_h2(b23 & 0xffffu));
        mma16816<MT>(o[4 * k + 3], pa, e4m3x2_to_h2(a23 >> 16), e4m3x2_to_h2(b23 >> 16));
      } else {
        mma16816<MT>(o[2 * k], pa, prmt(vraw[0][k], vraw[1][k], 0x5410), prmt(vraw[2][k], vraw[3][k], 0x5410));
        mma16816<MT>(o[2 * k + 1], pa, prmt(vraw[0][k], vraw[1][k], 0x7632), prmt(vraw[2][k], vraw[3][k], 0x7632));
      }
    }
    load_v(at_next);
    at = at_next;
    sk = sk_next;
    sv = sv_next;
  }

  // ---- fold the four warps ----
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (c == 0) {
      sM[warp][r + 8 * h] = m[h];
      sL[warp][r + 8 * h] = l[h];
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int d = (i / VW) * 8 * VW + (2 * c + e) * VW + i % VW;
      sO[warp][r][d] = o[i][e];
      sO[warp][r + 8][d] = o[i][2 + e];
    }
  __syncthreads();
  const int row = tid >> 3, d0 = (tid & 7) * (D / 8);
  if (row >= rows) return;
  const float mx = fmaxf(fmaxf(sM[0][row], sM[1][row]), fmaxf(sM[2][row], sM[3][row]));
  float f[4], den = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[k] = ex2(sM[k][row] - mx);
    den += f[k] * sL[k][row];
  }
  const float inv = den != 0.f ? 1.f / den : 0.f;
  const int qi = row / g, head = kvh * g + row % g;
  const int64_t dst_q = w.part_base < 0 ? w.q_begin + qi : w.part_base + qi;
#pragma unroll
  for (int d = d0; d < d0 + D / 8; d += 4) {
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
  if ((tid & 7) == 0) {
    const float lse = den > 0.f ? (mx + log2f(den)) * kLn2 : den == 0.f ? -INFINITY : den;
    // a NaN partial row is merged as +inf: the merge takes the maximum over its parts, which
    // passes over NaN, and inf - inf makes the row NaN there
    if (w.part_base >= 0)
      p.mid_lse[dst_q * p.hq + head] = den >= 0.f ? lse : INFINITY;
    else if (p.lse)
      p.lse[dst_q * p.hq + head] = lse;
  }
}

template <typename T, typename CT, int D>
static int paged_wide_launch(const PagedParams& p, int max_wide, cudaStream_t st);

template <typename T>
static int paged_launch(const PagedParams& p, bool q8, int D, int max_wide, int max_narrow,
                        int max_merge, cudaStream_t st) {
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
    auto go = [&](auto kernel) -> int {
      BE_CUDA_CHECK(launch_pdl(kernel, grid, dim3(128), 0, st, p));
      return BE_OK;
    };
    int rc;
    if (q8)
      rc = D == 128 ? go(paged_narrow_kernel<T, E4M3, 128>) : go(paged_narrow_kernel<T, E4M3, 64>);
    else
      rc = D == 128 ? go(paged_narrow_kernel<T, T, 128>) : go(paged_narrow_kernel<T, T, 64>);
    if (rc != BE_OK) return rc;
  }
  if (max_merge > 0) {
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

extern "C" int be_paged_attn_run(const int32_t* plan_dev, int max_wide, int max_narrow,
                                 int max_merge, int max_parts, int page_size, const void* q,
                                 int64_t q_row_stride, const void* paged_kv_cache,
                                 const float* kv_scale, int num_pages, int num_qo_heads,
                                 int num_kv_heads, int head_dim, int dtype, int cache_dtype,
                                 float sm_scale, void* out, int64_t out_row_stride, float* lse,
                                 float* mid_o, float* mid_lse, void* stream) {
  if (max_wide < 0 || max_narrow < 0 || max_merge < 0 || max_parts < 0 || page_size < 1 ||
      num_pages < 1 || num_kv_heads < 1 || num_kv_heads > 1024 || num_qo_heads < 1 ||
      std::max(max_wide, max_narrow) > (1 << 20) ||
      num_qo_heads % num_kv_heads) {
    set_error("be_paged_attn_run: invalid shape");
    return BE_EINVAL;
  }
  if ((dtype != BE_BF16 && dtype != BE_F16) || (cache_dtype != BE_E4M3 && cache_dtype != dtype)) {
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
  if (!plan_dev || !q || !paged_kv_cache || !out || (max_parts > 0 && (!mid_o || !mid_lse)) ||
      (cache_dtype == BE_E4M3) != (kv_scale != nullptr)) {
    set_error("be_paged_attn_run: null pointer (an 8-bit cache needs kv_scale, another has none)");
    return BE_EINVAL;
  }
  if (((uintptr_t)q | (uintptr_t)paged_kv_cache | (uintptr_t)mid_o) % 16 || (uintptr_t)out % 8 ||
      q_row_stride % 8 || out_row_stride % 4) {
    set_error("be_paged_attn_run: q and the cache must be 16-byte aligned, out 8-byte");
    return BE_EINVAL;
  }
  PagedParams p;
  p.plan = plan_dev;
  p.q = (const char*)q;
  p.q_row_stride = q_row_stride;
  p.pool = (const char*)paged_kv_cache;
  p.scale = kv_scale;
  p.num_pages = num_pages;
  p.ps = page_size;
  p.hq = num_qo_heads;
  p.hkv = num_kv_heads;
  p.g = num_qo_heads / num_kv_heads;
  p.scale_log2 = sm_scale * kLog2e;
  p.out = (char*)out;
  p.out_row_stride = out_row_stride;
  p.lse = lse;
  p.mid_o = mid_o;
  p.mid_lse = mid_lse;
  const bool q8 = cache_dtype == BE_E4M3;
  return dtype == BE_BF16
             ? paged_launch<__nv_bfloat16>(p, q8, head_dim, max_wide, max_narrow, max_merge, (cudaStream_t)stream)
             : paged_launch<__half>(p, q8, head_dim, max_wide, max_narrow, max_merge, (cudaStream_t)stream);
}
