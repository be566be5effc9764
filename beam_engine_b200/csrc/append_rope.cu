// Append to a paged cache with the position rotation on the way, into 8-bit
// (e4m3) pages with one scale per block or into pages of the rows' own type,
// and the read-back of 8-bit pages as values.
//
// A block is one page x plane (K | V) x KV head.  Its scale is a power of two,
//   e = the smallest integer in [-40, 40] with amax <= 448 * 2^e,
// over the block's finite new values, and never below the scale the block had,
// unless the call writes the page's slot 0, which begins the block anew.  With
// powers of two the scale costs no precision (e4m3 keeps 4 significant bits at
// every exponent, so up to one binary order less head room only moves where
// the subnormals begin), multiplying by it is exact, and tokens re-rounded when a
// later append raises the scale change only where they fall below the new
// subnormal step.  [-40, 40] keeps 1 / s and ratios of scales far inside fp32.
//
// Work split: a scale depends on every row that the call puts into its page, so
// one CTA owns a page's K and one its V.  Rows of a page are usually adjacent (a prompt) or alone
// (a beam step); a CTA takes the runs of equal pages that start inside its span
// of rows and looks for other runs of the same page anywhere in the call; the
// CTA of the first such run does the page, so rows may come in any order.  Up to
// ROPE_SCAN_ROWS rows a CTA compares every row's page itself.  Above that a
// first launch resolves the pages and lists the run starts per 256 rows with their pages, and
// the search reads only those lists (a 16th of the rows for a prompt with pages of 16).
//
// A warp takes one block's rows (up to 16 at a time) into registers, rotates them there, and has both
// the largest value and the codes from one read.  The rotation is done in 64 bits and rounded
// once: a value next to a border between two codes, or a block's largest next to one between
// two scales, then falls where the exact product does (fp32 left 5e-5 of a prompt's
// values one code off).
//
// Bound: HBM (rows in, codes out) for prompts; latency for a beam step.  8 prompts of 1024 rows, 8 KV heads of
// 128, bf16: 37 us (1.4 TB/s; the chain of a CTA's 16 rows, 64-bit conversions, 2 CTAs per SM
// by registers); 128 rows of a step: 5.4 us.  Reading 8192 tokens back as values: 10.7 us.
#include "common.cuh"

namespace be {

constexpr int ROPE_SCAN_ROWS = 512;   // largest call whose CTAs scan all rows
constexpr int ROPE_BLOCK = 256;       // rows per run-start list of the first launch
constexpr int ROPE_MAX_PAGE = 256;    // slots of a page (shared row table)
constexpr int ROPE_TAB = 16;          // rows whose cos / sin are in shared memory at once
constexpr int ROPE_SPAN = 16;         // rows of a CTA in a large call
constexpr float kE4M3Max = 448.f;
constexpr int kScaleExpMin = -40, kScaleExpMax = 40;

struct RopeAppend {
  const char* k;
  const char* v;
  int64_t k_stride, v_stride;       // elements between rows
  char* q;                          // fused rows whose q heads are rotated in place, or null
  int64_t q_stride;
  int hq;
  const int32_t* batch;             // null: write_page / write_pos name the slots directly
  const int32_t* pos;               // positions in the sequence (slots come from them with batch)
  const int32_t* rope_pos;          // positions of the rotation
  const int32_t* kv_indices;
  const int32_t* kv_indptr;
  const int32_t* write_page;
  const int32_t* write_pos;
  const float* inv_freq;            // null: no rotation
  char* cache;
  float* scale;                     // [pages][2][hkv]; null: cache of the rows' type
  int n, num_pages, ps, hkv, D, span;
  int32_t* page_of;                 // workspace of the first launch: [n] pages,
  int32_t* slot_of;                 // [n] slots,
  int2* starts;                     // [ceil(n / 256)][256] run starts: row, page
  int32_t* n_starts;                // [ceil(n / 256)]
};

__device__ __forceinline__ void rope_slot(const RopeAppend& a, int i, int& page, int& slot) {
  if (a.batch) {
    const int pos = a.pos[i];
    const int b = a.batch[i];
    page = -1;
    slot = 0;
    if (pos >= 0) {
      page = a.kv_indices[a.kv_indptr[b] + pos / a.ps];
      slot = pos % a.ps;
    }
  } else {
    page = a.write_page[i];
    slot = a.write_pos[i];
  }
  if (page < 0 || page >= a.num_pages || slot < 0 || slot >= a.ps) page = -1;
}

// Smallest e in [-40, 40] with amax <= 448 * 2^e (448 = 1.75 * 2^8), read off the
// exponent and mantissa bits; amax is finite and >= 0.
__device__ __forceinline__ float block_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = min(max(e, kScaleExpMin), kScaleExpMax);   // amax = 0 and subnormals: -40
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// two e4m3 codes (low byte first) -> two halves, exactly
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}
__device__ __forceinline__ void e4m3x4_to_f(uint32_t w, float* f) {
  const uint32_t a = e4m3x2_to_h2(w & 0xffffu), b = e4m3x2_to_h2(w >> 16);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a));
  const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&b));
  f[0] = x.x; f[1] = x.y; f[2] = y.x; f[3] = y.y;
}

// First launch of a call with many rows: page and slot of every row, and per 256
// rows the list of rows whose page differs from the row before.
__global__ void __launch_bounds__(ROPE_BLOCK) rope_runs_kernel(const RopeAppend a) {
  __shared__ int count;
  pdl_wait();
  pdl_trigger();   // the append launch waits for this grid before it reads the lists
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  const int i = blockIdx.x * ROPE_BLOCK + threadIdx.x;
  if (i < a.n) {
    int page, slot, before = -1, s2;
    rope_slot(a, i, page, slot);
    if (i > 0) rope_slot(a, i - 1, before, s2);
    a.page_of[i] = page;
    a.slot_of[i] = slot;
    if (page < 0) flag_range_error();
    if (page >= 0 && (i == 0 || before != page))
      a.starts[blockIdx.x * ROPE_BLOCK + atomicAdd(&count, 1)] = make_int2(i, page);
  }
  __syncthreads();
  if (threadIdx.x == 0) a.n_starts[blockIdx.x] = count;
}

// cos / sin of rows rows[0..m) into the table.  The angle is a product of two fp32
// numbers in 64 bits, reduced to turns there: the rounding of an fp32 product
// alone is 6e-3 rad at position 100 000.  A lane rotates dims 8 j .. 8 j + 7 of its row one after
// the other, so entry (row, i, j) holds dim 8 j + i: neighbouring lanes read neighbouring entries.
template <typename F2>
__device__ __forceinline__ void rope_table(const RopeAppend& a, const int* rows, int m, int half,
                                           F2* tab) {
  for (int i = threadIdx.x; i < m * half; i += blockDim.x) {
    const int lp = half / 8, r = i / half, e = i - r * half, d = 8 * (e % lp) + e / lp;
    const double turns = (double)a.rope_pos[rows[r]] * (double)a.inv_freq[d] * 0.15915494309189535;
    const double t = 2.0 * (turns - rint(turns));
    if constexpr (std::is_same<F2, double2>::value) {
      double s, c;
      sincospi(t, &s, &c);
      tab[i] = make_double2(c, s);
    } else {
      float s, c;
      sincospif((float)t, &s, &c);
      tab[i] = make_float2(c, s);
    }
  }
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float* f) {
  if constexpr (sizeof(T) == 2) {
    if (vec) {
      const int4 raw = *reinterpret_cast<const int4*>(p);
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = to_f(e[i]);
      return;
    }
  } else if (vec) {
    const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
    f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w;
    f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f(p[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, const float* f) {
  if (vec) {
    if constexpr (sizeof(T) == 2) {
      int4 raw;
      T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = from_f<T>(f[i]);
      *reinterpret_cast<int4*>(p) = raw;
    } else {
      reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] = from_f<T>(f[i]);
}

// Eight dims of each half of one row: dims [8 j, 8 j + 8) in lo, those + D/2 in hi, rotated
// by the row's table entry.
__device__ __forceinline__ void rope_rotate(const double2* tab, int j, int lp, float* lo, float* hi) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double2 cs = tab[i * lp + j];
    const double x = lo[i], y = hi[i];
    lo[i] = (float)(x * cs.x - y * cs.y);
    hi[i] = (float)(y * cs.x + x * cs.y);
  }
}

__device__ __forceinline__ float finite_abs(float x) {   // 0 for infinities and NaN
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// Rows of the page that a warp holds at once: ITS instructions of 32 / (D / 16) rows.
constexpr int ROPE_ITS = 4;

template <typename T, bool QUANT>
__global__ void __launch_bounds__(256) rope_append_kernel8(const RopeAppend a) {
  extern __shared__ double2 tab[];                 // [ROPE_TAB][D / 2]
  __shared__ int row_of[ROPE_MAX_PAGE];            // slot -> row of the call (the last one), or -1
  __shared__ int list[ROPE_MAX_PAGE];              // slots of the page with rows, in order
  __shared__ float amax_s[64];                     // per head: hkv <= 64
  __shared__ int batch_rows[ROPE_TAB];
  __shared__ int span_page[ROPE_SPAN + 1];         // pages of the row before the span and of its rows
  __shared__ int n_list, first;
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int D = a.D, half = D / 2, lp = D / 16;    // lanes per row: 8 + 8 dims each
  const bool listed = a.page_of != nullptr;
  const int i0 = blockIdx.x * a.span, i1 = min(a.n, i0 + a.span);
  const int tpw = 32 / lp;                         // rows per warp instruction
  const int j = lane % lp, sub = lane / lp;
  const int plane = blockIdx.y;                    // K, or V and the q heads
  const T* rows_in = reinterpret_cast<const T*>(plane ? a.v : a.k);
  const int64_t stride_in = plane ? a.v_stride : a.k_stride;
  const bool vec = ((((uintptr_t)rows_in) | (stride_in * sizeof(T))) & 15) == 0;
  const bool rotate = !plane && a.inv_freq;
  if (tid <= i1 - i0) {
    int pg = -1, s2;
    const int r = i0 - 1 + tid;
    if (listed) {
      if (r >= 0) pg = a.page_of[r];
    } else if (r >= 0) {
      rope_slot(a, r, pg, s2);
      if (pg < 0 && tid > 0 && plane == 0) flag_range_error();
    }
    span_page[tid] = pg;
  }
  __syncthreads();

  // ---- q heads of the span's rows, rotated in place ----
  if (a.q && plane == 1) {
    float2* qtab = reinterpret_cast<float2*>(tab);
    const bool vec_q = ((((uintptr_t)a.q) | (a.q_stride * sizeof(T))) & 15) == 0;
    for (int b0 = i0; b0 < i1; b0 += ROPE_TAB) {
      const int m = min(ROPE_TAB, i1 - b0);
      __syncthreads();
      if (tid < m) list[tid] = b0 + tid;
      __syncthreads();
      rope_table(a, list, m, half, qtab);
      __syncthreads();
      for (int u = tid / lp; u < m * a.hq; u += blockDim.x / lp) {
        const int r = u / a.hq, h = u - r * a.hq;
        T* dst = reinterpret_cast<T*>(a.q) + (b0 + r) * a.q_stride + (int64_t)h * D;
        float lo[8], hi[8];
        load8<T>(dst + 8 * j, vec_q, lo);
        load8<T>(dst + 8 * j + half, vec_q, hi);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 cs = qtab[r * half + i * lp + j];
          const float x = lo[i], y = hi[i];
          lo[i] = x * cs.x - y * cs.y;
          hi[i] = y * cs.x + x * cs.y;
        }
        store8<T>(dst + 8 * j, vec_q, lo);
        store8<T>(dst + 8 * j + half, vec_q, hi);
      }
    }
  }

  for (int i = i0; i < i1; ++i) {
    // ---- does a run of rows of one page start here? ----
    const int page = span_page[i - i0 + 1];
    if (page < 0 || span_page[i - i0] == page) continue;     // uniform over the CTA
    // ---- rows of the call that go into this page, and the first of them ----
    __syncthreads();
    for (int s = tid; s < a.ps; s += blockDim.x) row_of[s] = -1;
    if (tid == 0) {
      first = a.n;
      n_list = 0;
    }
    __syncthreads();
    if (listed) {
      const int nb = (a.n + ROPE_BLOCK - 1) / ROPE_BLOCK;
      const int per = nb < (int)blockDim.x ? blockDim.x / nb : 1;   // threads per list
      for (int b = tid / per; b < nb; b += blockDim.x / per) {
        const int m = a.n_starts[b];
        for (int k = tid % per; k < m; k += per) {
          const int2 start = a.starts[b * ROPE_BLOCK + k];
          if (start.y != page) continue;
          atomicMin(&first, start.x);
          const int at = atomicAdd(&n_list, 1);
          if (at < ROPE_MAX_PAGE) list[at] = start.x;
        }
      }
      __syncthreads();
      if (first != i) continue;                   // another CTA (or run) has the page
      // the runs' rows, a thread each; a page written more often than it has slots is looked up whole
      const int runs = n_list <= ROPE_MAX_PAGE ? n_list : 1;
      for (int k = 0; k < runs; ++k) {
        const int start = n_list <= ROPE_MAX_PAGE ? list[k] : i;
        for (int r0 = start; r0 < a.n; r0 += blockDim.x) {
          const int r = r0 + tid;
          const bool hit = r < a.n && a.page_of[r] == page;
          if (hit) atomicMax(&row_of[a.slot_of[r]], r);
          const bool on = __syncthreads_or(tid == (int)blockDim.x - 1 && hit);
          if (!on && n_list <= ROPE_MAX_PAGE) break;
        }
      }
    } else {
      for (int r = tid; r < a.n; r += blockDim.x) {
        int p, s;
        rope_slot(a, r, p, s);
        if (p != page) continue;
        atomicMin(&first, r);
        atomicMax(&row_of[s], r);
      }
    }
    __syncthreads();
    if (first != i) continue;                     // another CTA (or run) has the page
    if (warp == 0) {                              // compact, in slot order
      int m = 0;
      for (int s0 = 0; s0 < a.ps; s0 += 32) {
        const int s = s0 + lane;
        const int r = s < a.ps ? row_of[s] : -1;
        const unsigned has = __ballot_sync(0xffffffffu, r >= 0);
        if (r >= 0) list[m + __popc(has & ((1u << lane) - 1))] = s;
        m += __popc(has);
      }
      if (lane == 0) n_list = m;
    }
    __syncthreads();
    const int m = n_list;
    const bool fresh = row_of[0] >= 0;
    const int64_t plane_rows = (int64_t)a.ps * a.hkv;
    // Rows go by batches of ROPE_TAB (the table's size).  A page of one batch (of any length that
    // its table and a warp's registers hold) is read once: largest value, scale, codes.  More
    // batches are walked twice, first for the scale.
    const int n_batch = (m + ROPE_TAB - 1) / ROPE_TAB;
    const int held = ROPE_ITS * tpw;              // rows that a warp holds
    const bool once = m <= min(held, ROPE_TAB);
    auto load_batch = [&](int b) {
      const int c0 = b * ROPE_TAB, cm = min(ROPE_TAB, m - c0);
      __syncthreads();
      if (tid < cm) batch_rows[tid] = row_of[list[c0 + tid]];
      __syncthreads();
      if (rotate) {
        rope_table(a, batch_rows, cm, half, tab);
        __syncthreads();
      }
      return cm;
    };
    // the block's new scale; where it grew, the tokens that were there get its steps
    auto new_scale = [&](int h, float amax) -> float {
      float* sp = a.scale + ((int64_t)page * 2 + plane) * a.hkv + h;
      const float old = fresh ? 0.f : *sp;
      const float s = fmaxf(block_scale(amax), old);
      __syncwarp();
      if (lane == 0) *sp = s;
      if (fresh || !(s > old)) return s;
      const float ratio = old / s;                // a power of two, or 0 for a block never written
      const int words = D / 4;
      for (int w = lane; w < a.ps * words; w += 32) {
        const int sl = w / words;
        if (row_of[sl] >= 0) continue;            // this call writes it
        uint32_t* p = reinterpret_cast<uint32_t*>(
            a.cache + (((int64_t)page * 2 + plane) * plane_rows + (int64_t)sl * a.hkv + h) * D) +
            (w - sl * words);
        float f[4];
        e4m3x4_to_f(*p, f);
        *p = to_e4m3x2(f[0] * ratio, f[1] * ratio) | to_e4m3x2(f[2] * ratio, f[3] * ratio) << 16;
      }
      return s;
    };
    // rows [t0, t0 + held) of the batch into registers; codes (or values) from there
    auto take = [&](int h, int t0, int cm, float (&lo)[ROPE_ITS][8], float (&hi)[ROPE_ITS][8]) -> float {
      float best = 0.f;
#pragma unroll
      for (int it = 0; it < ROPE_ITS; ++it) {
        const int t = t0 + it * tpw + sub;
        if (t < cm) {
          const T* src = rows_in + batch_rows[t] * stride_in + (int64_t)h * D + 8 * j;
          load8<T>(src, vec, lo[it]);
          load8<T>(src + half, vec, hi[it]);
        }
      }
#pragma unroll
      for (int it = 0; it < ROPE_ITS; ++it) {
        const int t = t0 + it * tpw + sub;
        if (t >= cm) continue;
        if (rotate) rope_rotate(tab + t * half, j, lp, lo[it], hi[it]);
#pragma unroll
        for (int k = 0; k < 8; ++k) best = fmaxf(best, fmaxf(finite_abs(lo[it][k]), finite_abs(hi[it][k])));
      }
      return best;
    };
    auto put = [&](int h, int c0, int t0, int cm, float s, const float (&lo)[ROPE_ITS][8],
                   const float (&hi)[ROPE_ITS][8]) {
      const float inv = 1.f / s;                  // exact: a power of two
#pragma unroll
      for (int it = 0; it < ROPE_ITS; ++it) {
        const int t = t0 + it * tpw + sub;
        if (t >= cm) continue;
        const int64_t row = ((int64_t)page * 2 + plane) * plane_rows + (int64_t)list[c0 + t] * a.hkv + h;
        if constexpr (QUANT) {
          char* dst = a.cache + row * D + 8 * j;
          const float* x = lo[it];
          const float* y = hi[it];
          uint2 cl, ch;
          cl.x = to_e4m3x2(x[0] * inv, x[1] * inv) | to_e4m3x2(x[2] * inv, x[3] * inv) << 16;
          cl.y = to_e4m3x2(x[4] * inv, x[5] * inv) | to_e4m3x2(x[6] * inv, x[7] * inv) << 16;
          ch.x = to_e4m3x2(y[0] * inv, y[1] * inv) | to_e4m3x2(y[2] * inv, y[3] * inv) << 16;
          ch.y = to_e4m3x2(y[4] * inv, y[5] * inv) | to_e4m3x2(y[6] * inv, y[7] * inv) << 16;
          *reinterpret_cast<uint2*>(dst) = cl;
          *reinterpret_cast<uint2*>(dst + half) = ch;
        } else {
          T* dst = reinterpret_cast<T*>(a.cache) + row * D + 8 * j;
          const bool vec_c = ((uintptr_t)a.cache & 15) == 0;
          store8<T>(dst, vec_c, lo[it]);
          store8<T>(dst + half, vec_c, hi[it]);
        }
      }
    };
    auto warp_max = [&](float x) {
#pragma unroll
      for (int off = 16; off; off >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
      return x;
    };
    float lo[ROPE_ITS][8], hi[ROPE_ITS][8];
    if (once || !QUANT) {
      for (int b = 0; b < n_batch; ++b) {
        const int cm = load_batch(b);
        for (int h = warp; h < a.hkv; h += warps)
          for (int t0 = 0; t0 < cm; t0 += held) {
            const float best = take(h, t0, cm, lo, hi);
            float s = 1.f;
            if constexpr (QUANT) s = new_scale(h, warp_max(best));
            put(h, b * ROPE_TAB, t0, cm, s, lo, hi);
          }
      }
    } else {
      for (int h = tid; h < a.hkv; h += blockDim.x) amax_s[h] = 0.f;
      for (int b = 0; b < n_batch; ++b) {
        const int cm = load_batch(b);
        for (int h = warp; h < a.hkv; h += warps)
          for (int t0 = 0; t0 < cm; t0 += held) {
            const float best = warp_max(take(h, t0, cm, lo, hi));
            __syncwarp();
            if (lane == 0) amax_s[h] = fmaxf(amax_s[h], best);   // only this warp has head h
          }
      }
      __syncthreads();
      for (int h = warp; h < a.hkv; h += warps) {
        const float s = new_scale(h, amax_s[h]);
        __syncwarp();
        if (lane == 0) amax_s[h] = s;
      }
      for (int b = 0; b < n_batch; ++b) {
        const int cm = load_batch(b);
        for (int h = warp; h < a.hkv; h += warps)
          for (int t0 = 0; t0 < cm; t0 += held) {
            take(h, t0, cm, lo, hi);
            put(h, b * ROPE_TAB, t0, cm, amax_s[h], lo, hi);
          }
      }
    }
  }
}

// Pages of an 8-bit cache as the values they stand for: out [n][2][ps][hkv][D].  A CTA
// per (page, plane), 16 codes per load, a thread's loads all before its first store.
template <typename T>
__global__ void __launch_bounds__(256) read_pages_kernel(const char* __restrict__ cache,
                                                         const float* __restrict__ scale,
                                                         const int32_t* __restrict__ pages,
                                                         int num_pages, int ps, int hkv, int D,
                                                         T* __restrict__ out) {
  __shared__ float sc[64];
  pdl_wait();
  const int pg = blockIdx.x >> 1, plane = blockIdx.x & 1, page = pages[pg];
  const bool has = page >= 0 && page < num_pages;
  if (!has && threadIdx.x == 0 && plane == 0) flag_range_error();
  for (int h = threadIdx.x; h < hkv; h += blockDim.x)
    sc[h] = has ? scale[((int64_t)page * 2 + plane) * hkv + h] : 0.f;
  __syncthreads();
  const int vecs = ps * hkv * D / 16, per_row = D / 16;
  const int4* src = reinterpret_cast<const int4*>(cache) + ((int64_t)max(page, 0) * 2 + plane) * vecs;
  T* dst = out + ((int64_t)pg * 2 + plane) * vecs * 16;
  constexpr int U = 4;
  for (int i0 = threadIdx.x; i0 < vecs; i0 += 256 * U) {
    int4 c[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      c[u] = has && i0 + 256 * u < vecs ? __ldg(src + i0 + 256 * u) : make_int4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + 256 * u;
      if (i >= vecs) break;
      const float s = sc[(i / per_row) % hkv];
      const uint32_t w[4] = {(uint32_t)c[u].x, (uint32_t)c[u].y, (uint32_t)c[u].z, (uint32_t)c[u].w};
      float f[16];
#pragma unroll
      for (int k = 0; k < 4; ++k) e4m3x4_to_f(w[k], f + 4 * k);
#pragma unroll
      for (int k = 0; k < 16; ++k) f[k] *= s;
      store8<T>(dst + (int64_t)i * 16, true, f);
      store8<T>(dst + (int64_t)i * 16 + 8, true, f + 8);
    }
  }
}

static int rope_append_launch(RopeAppend& a, int dtype, int32_t* workspace, cudaStream_t st) {
  // one row per CTA while that is what fills the GPU (a beam step), pages' worth of rows
  // once there are many: the search for other runs is then shared by a CTA's rows
  a.span = a.n <= ROPE_SCAN_ROWS ? 1 : ROPE_SPAN;
  if (a.n > ROPE_SCAN_ROWS) {
    const int nb = (a.n + ROPE_BLOCK - 1) / ROPE_BLOCK;
    a.page_of = workspace;
    a.slot_of = a.page_of + a.n;
    a.n_starts = a.slot_of + a.n;
    a.starts = reinterpret_cast<int2*>(workspace + (2 * (int64_t)a.n + nb + 1) / 2 * 2);
    BE_CUDA_CHECK(launch_pdl(rope_runs_kernel, dim3(nb), dim3(ROPE_BLOCK), 0, st, a));
  }
  const dim3 grid((a.n + a.span - 1) / a.span, 2);
  const size_t smem = (size_t)ROPE_TAB * (a.D / 2) * sizeof(double2);   // <= 32 KB
#define BE_ROPE8(T)                                                                            \
  do {                                                                                         \
    if (a.scale)                                                                               \
      BE_CUDA_CHECK(launch_pdl(rope_append_kernel8<T, true>, grid, dim3(256), smem, st, a));   \
    else                                                                                       \
      BE_CUDA_CHECK(launch_pdl(rope_append_kernel8<T, false>, grid, dim3(256), smem, st, a));  \
  } while (0)
  switch (dtype) {
    case BE_BF16: BE_ROPE8(__nv_bfloat16); break;
    case BE_F16: BE_ROPE8(__half); break;
    default: BE_ROPE8(float);
  }
#undef BE_ROPE8
  BE_LAUNCH_CHECK();
  return BE_OK;
}

static int rope_append_check(const char* fn, const RopeAppend& a, int dtype, int cache_dtype,
                             const int32_t* workspace, int64_t workspace_ints) {
  const int D = a.D;
  if (a.n < 0 || a.num_pages < 1 || a.ps < 1 || a.ps > ROPE_MAX_PAGE || a.hkv < 1 || a.hkv > 64 ||
      dtype < BE_F32 || dtype > BE_BF16 || (cache_dtype != BE_E4M3 && cache_dtype != dtype)) {
    set_error("%s: invalid shape or type (page size 1..%d, kv heads 1..64, cache e4m3 or of the rows' type)",
              fn, ROPE_MAX_PAGE);
    return BE_EINVAL;
  }
  if (D != 32 && D != 64 && D != 128 && D != 256) {
    set_error("%s: head_dim %d is not 32, 64, 128 or 256", fn, D);
    return BE_EINVAL;
  }
  if (a.n == 0) return BE_OK;
  if (!a.k || !a.v || !a.cache || (cache_dtype == BE_E4M3) != (a.scale != nullptr) ||
      (!a.batch && (!a.write_page || !a.write_pos)) ||
      (a.batch && (!a.pos || !a.kv_indices || !a.kv_indptr)) || (a.inv_freq && !a.rope_pos)) {
    set_error("%s: null pointer (an 8-bit cache needs kv_scale, another cache has none)", fn);
    return BE_EINVAL;
  }
  if (cache_dtype == BE_E4M3 && (uintptr_t)a.cache % 8) {
    set_error("%s: the cache must be 8-byte aligned", fn);
    return BE_EINVAL;
  }
  if (a.n > ROPE_SCAN_ROWS && (!workspace || workspace_ints < 5ll * a.n + 1024)) {
    set_error("%s: %d rows need a workspace of %lld ints", fn, a.n, 5ll * a.n + 1024);
    return BE_ECAPACITY;
  }
  if (a.n > ROPE_SCAN_ROWS && (uintptr_t)workspace % 8) {
    set_error("%s: the workspace must be 8-byte aligned", fn);
    return BE_EINVAL;
  }
  return BE_OK;
}

}  // namespace be

using namespace be;

extern "C" int be_rope_append_paged_kv(const be_rope_append_args* args) {
  if (!args) {
    set_error("be_rope_append_paged_kv: null pointer");
    return BE_EINVAL;
  }
  const be_rope_append_args& g = *args;
  RopeAppend a{};
  a.k = (const char*)g.append_key;
  a.v = (const char*)g.append_value;
  a.k_stride = g.key_row_stride;
  a.v_stride = g.value_row_stride;
  a.batch = g.batch_indices;
  a.pos = g.positions;
  a.rope_pos = g.rope_positions ? g.rope_positions : g.positions;
  a.kv_indices = g.kv_indices;
  a.kv_indptr = g.kv_indptr;
  a.inv_freq = g.inv_freq;
  a.cache = (char*)g.paged_kv_cache;
  a.scale = g.kv_scale;
  a.n = g.nnz;
  a.num_pages = g.num_pages;
  a.ps = g.page_size;
  a.hkv = g.num_kv_heads;
  a.D = g.head_dim;
  if (a.n > 0 && !a.batch) {
    set_error("be_rope_append_paged_kv: null pointer");
    return BE_EINVAL;
  }
  const int rc = rope_append_check("be_rope_append_paged_kv", a, g.dtype, g.cache_dtype, g.workspace,
                                   g.workspace_ints);
  if (rc != BE_OK || a.n == 0) return rc;
  return rope_append_launch(a, g.dtype, g.workspace, (cudaStream_t)g.stream);
}

extern "C" int be_rope_qkv_append8(void* qkv, int64_t row_stride, int n, int num_qo_heads,
                                   int num_kv_heads, int head_dim, const int32_t* positions,
                                   const float* inv_freq, void* paged_kv_cache, float* kv_scale,
                                   int num_pages, int page_size, const int32_t* write_page,
                                   const int32_t* write_pos, int dtype, int32_t* workspace,
                                   int64_t workspace_ints, void* stream) {
  if (num_qo_heads < 0 || !inv_freq || !positions) {
    set_error("be_rope_qkv_append8: invalid shape or null pointer");
    return BE_EINVAL;
  }
  const int elt = dtype_size(dtype);
  RopeAppend a{};
  a.q = (char*)qkv;
  a.q_stride = a.k_stride = a.v_stride = row_stride;
  a.hq = num_qo_heads;
  a.k = (const char*)qkv + (int64_t)num_qo_heads * head_dim * elt;
  a.v = a.k + (int64_t)num_kv_heads * head_dim * elt;
  a.rope_pos = positions;
  a.write_page = write_page;
  a.write_pos = write_pos;
  a.inv_freq = inv_freq;
  a.cache = (char*)paged_kv_cache;
  a.scale = kv_scale;
  a.n = n;
  a.num_pages = num_pages;
  a.ps = page_size;
  a.hkv = num_kv_heads;
  a.D = head_dim;
  if (n > 0 && !qkv) {
    set_error("be_rope_qkv_append8: null pointer");
    return BE_EINVAL;
  }
  const int rc = rope_append_check("be_rope_qkv_append8", a, dtype, BE_E4M3, workspace, workspace_ints);
  if (rc != BE_OK || n == 0) return rc;
  return rope_append_launch(a, dtype, workspace, (cudaStream_t)stream);
}

extern "C" int be_read_paged_kv8(const void* paged_kv_cache, const float* kv_scale,
                                 const int32_t* pages, int n, int num_pages, int page_size,
                                 int num_kv_heads, int head_dim, void* out, int out_dtype,
                                 void* stream) {
  if (n < 0 || num_pages < 1 || page_size < 1 || page_size > ROPE_MAX_PAGE || num_kv_heads < 1 ||
      num_kv_heads > 64 || head_dim < 16 || head_dim > 256 || head_dim % 16 || out_dtype < BE_F32 ||
      out_dtype > BE_BF16 || n > (1 << 29)) {
    set_error("be_read_paged_kv8: invalid shape or dtype");
    return BE_EINVAL;
  }
  if (n == 0) return BE_OK;
  if (!paged_kv_cache || !kv_scale || !pages || !out || (uintptr_t)paged_kv_cache % 16 ||
      (uintptr_t)out % 16) {
    set_error("be_read_paged_kv8: null or misaligned pointer");
    return BE_EINVAL;
  }
  const dim3 grid((unsigned)n * 2);
  cudaStream_t st = (cudaStream_t)stream;
#define BE_READ8(T)                                                                            \
  BE_CUDA_CHECK(launch_pdl(read_pages_kernel<T>, grid, dim3(256), 0, st,                       \
                           (const char*)paged_kv_cache, kv_scale, pages, num_pages, page_size,     \
                           num_kv_heads, head_dim, (T*)out))
  switch (out_dtype) {
    case BE_BF16: BE_READ8(__nv_bfloat16); break;
    case BE_F16: BE_READ8(__half); break;
    default: BE_READ8(float);
  }
#undef BE_READ8
  BE_LAUNCH_CHECK();
  return BE_OK;
}
