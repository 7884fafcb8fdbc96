// Beam search over chains: the best continuations of all beams of an example, and the states that follow them.  The
// deterministic sibling of the multinomial / systematic resampling (cs_lair.hip, cs_final_resample).
//
// Selection.  s[k,v] = scores[k] + (logits[k,v] - lse[k]), lse the log of the sum of exponentials of the allowed logits
// of beam k: the W largest over (k,v), ties to the lowest k*V + v.  One pass over the logits: a wavefront holds a
// stretch of one beam in registers (LANE values per lane), leaves their sum of exponentials and those of them that can
// be among its W best in the workspace; a workgroup per example then joins the stretches of every beam, turns the
// kept logits into scores and takes the W best of them.  The normaliser joins before scores of different beams are
// compared, so within a beam a stretch's candidates can be chosen by their logits alone; where 64 bits give different logits
// one score, what such a choice left out is looked for once more (bm_join).  Sums and scores are held in
// 64 bits: two beams' candidates are often closer than float32 sums of 10^5 terms are exact, and the indices are to be
// those of the definition.
#include "cs_common.h"
#include "cs_div.h"
#include <type_traits>

namespace {

constexpr int BM_MAXW = 64;            // candidates per example: a lane each
constexpr int BM_MAXK = 2048;
constexpr int BM_JOIN = 1024;          // threads that join an example, at most
constexpr int BM_ONE = 8;              // stretches of an example, at most, for one launch that does it all
constexpr float BM_LOWEST = -3.402823466e+38f;

// of a stretch: the sum of exp(x - ref), ref being the largest logit or 0; the largest logit; the bound that all kept ones reach and
// no others do; the number of kept ones.  NaN in the place of the bound: some that equal the last kept one were not kept, and
// the largest of the smaller ones stands behind it in the list.
struct BmStat { double sum; float ref, top, cut; int32_t n; };

struct BmArgs {
  cs_beam_cfg c;
  const void *scores, *logits;
  const uint8_t *mask, *finished;
  BmStat* stat;     // [B*K*stretches]
  float* item_x;    // [B*K*stretches][keep] the logits kept of a stretch
  int32_t* item_v;  // and their values
  void* out_scores;
  int64_t *parents, *tokens;
  int32_t stretches, keep, len;   // values of a stretch
  uint32_t items;          // B*K*stretches
  CsDiv by_stretches, by_K, by_keep;
};

// The kernel's arguments, read anew: without this those that one part of a kernel alone needs are loaded at its start and kept, or
// spilled, to there.
__device__ __forceinline__ const BmArgs& bm_args() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();   // (they are the first ones)
  asm volatile("" : "+s"(p));
  return *(const BmArgs*)p;
}

__device__ __forceinline__ uint32_t bm_key(float v) {
  const uint32_t u = __float_as_uint(v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float bm_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ uint64_t bm_key64(double v) {   // 0: no candidate (NaN or -inf)
  if (!(v > -__builtin_inf())) return 0;
  const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);   // (+ 0.0: one zero)
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double bm_value64(uint64_t k) {
  return __longlong_as_double((long long)((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k));
}

template <typename T> struct BmElem;
template <> struct BmElem<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void widen(const uint32_t* r, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r[i]);
  }
};
struct BmBf16 { uint16_t u; };
template <> struct BmElem<BmBf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void widen(const uint32_t* r, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(r[i] << 16);
      x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  }
};
template <> struct BmElem<_Float16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void widen(const uint32_t* r, float* x) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const h2 h = __builtin_bit_cast(h2, r[i]);
      x[2 * i] = (float)h.x;
      x[2 * i + 1] = (float)h.y;
    }
  }
};

// Reductions by DPP moves within and across the rows of 16 lanes; lane 63 ends with the result of all.
template <int CTRL, int ROWS>
__device__ __forceinline__ int bm_dpp(int old, int v) {
  return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xf, false);
}
constexpr int BM_SHR = 0x110, BM_BCAST15 = 0x142, BM_BCAST31 = 0x143;
__device__ __forceinline__ float bm_wave_max(float v) {
#define CS_STEP(CTRL_, ROWS_) v = fmaxf(v, __int_as_float(bm_dpp<CTRL_, ROWS_>(__float_as_int(v), __float_as_int(v))));
  CS_STEP(BM_SHR + 1, 0xf) CS_STEP(BM_SHR + 2, 0xf) CS_STEP(BM_SHR + 4, 0xf) CS_STEP(BM_SHR + 8, 0xf)
  CS_STEP(BM_BCAST15, 0xa) CS_STEP(BM_BCAST31, 0xc)
#undef CS_STEP
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ double bm_wave_sum(double v) {
#define CS_STEP(CTRL_, ROWS_) \
  v += __hiloint2double(bm_dpp<CTRL_, ROWS_>(0, __double2hiint(v)), bm_dpp<CTRL_, ROWS_>(0, __double2loint(v)));
  CS_STEP(BM_SHR + 1, 0xf) CS_STEP(BM_SHR + 2, 0xf) CS_STEP(BM_SHR + 4, 0xf) CS_STEP(BM_SHR + 8, 0xf)
  CS_STEP(BM_BCAST15, 0xa) CS_STEP(BM_BCAST31, 0xc)
#undef CS_STEP
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), 63), __builtin_amdgcn_readlane(__double2loint(v), 63));
}

// 2^(j / 64)
__device__ const double bm_pow64[64] = {
    1, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.1023825833078409, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.2021567314527031, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.2553807570246911, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.3396675240533029,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.5590044002378369, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.6457554781539649, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.7186192981224779, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.9784560263879509};

// exp(d) for |d| <= 690 as 2^n 2^(j/64) exp(r), 64 n + j the integer nearest to 64 d / ln 2 and |r| <= ln 2 / 128, exp(r) by its
// Taylor polynomial of degree 4 (remainder r^5 / 120 < 4e-14; degree 3, 3.6e-11, would be 3 us faster on the largest case and
// mistakes the order of beams that are certain to 1e-11): the table-driven method of Tang (1989).  Adding 1.5 * 2^52
// leaves the integer in the low word.  The table lies in the lanes' registers and is read by ds_bpermute, which takes the
// lane (all of them have to be there) from the index's low 6 bits by itself; its high words have j << 14 taken off beforehand, so one shift and addition of
// the whole integer puts the exponent right.
struct BmPow {
  int hi, lo;
  __device__ __forceinline__ explicit BmPow(int lane) {
    const double t = bm_pow64[lane];
    hi = __double2hiint(t) - (lane << 14);
    lo = __double2loint(t);
  }
};
__device__ __forceinline__ double bm_add_exp(double sum, double d, const BmPow& pow) {
  constexpr double MAGIC = 6755399441055744.0;
  const double z = __builtin_fma(d, 92.33248261689366, MAGIC);
  const int nj = __double2loint(z);
  const double r = __builtin_fma(z - MAGIC, -0.010830424696249145, d);
  const int hi = __builtin_amdgcn_ds_bpermute(nj << 2, pow.hi) + (nj << 14), lo = __builtin_amdgcn_ds_bpermute(nj << 2, pow.lo);
  const double p = __builtin_fma(__builtin_fma(__builtin_fma(__builtin_fma(r, 1.0 / 24, 1.0 / 6), r, 0.5), r, 1.0), r, 1.0);
  return __builtin_fma(__hiloint2double(hi, lo), p, sum);
}

// The largest key, as far as its leading BITS bits say, that at least W lanes reach with theirs; 0 if fewer than W lanes
// have one.  A bound that is a little low only lets a few more candidates through.
template <int BITS>
__device__ __forceinline__ uint32_t bm_wave_threshold(uint32_t key, int W) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = 31; bit > 31 - BITS; --bit) {
    const uint32_t u = t | (1u << bit);
    if (__popcll(__ballot(key >= u)) >= W) t = u;
  }
  return t;
}

// One wavefront per stretch.  Bound by vector instructions where the logits have 16 bits: 619 of them for 2048 values, 364 of
// these the 64-bit exponentials (91 for 8 values of a lane); 64 x 16 rows of 131072 bfloat16 (268 MB) take 82 to 90 us, 81 % of the
// launch's cycles issuing them, where their bytes alone would take 45.  In float32 it is bound by memory: 4096 rows of 10200 (167 MB)
// take 33 to 38 us, 4.4 to 5.1 TB/s.  A value below -690 sends its stretch through the exponentials again: 103 -> 157 us with a third at -inf.
// (Logits and values kept in two arrays, so that a kept one costs 4 instructions and not 8: 3 % faster.)
// 32 values per lane measured 104 us there against 115 (16), 147 (8) and 164 (64: too few wavefronts fit); asking for the
// next stretch before working on one (a fixed set of wavefronts) measured 141: twice the registers.
template <typename T, bool MASK, int LANE>
__device__ __forceinline__ void bm_scan(const BmArgs& a, uint32_t row, uint32_t stretch, BmStat* stat, float* out_x, int32_t* out_v) {
  constexpr int N = BmElem<T>::N;      // logits in 16 bytes
  constexpr float INF = __builtin_inff();
  const int lane = threadIdx.x & 63;
  const int32_t base = (int32_t)stretch * (64 * LANE);
  const uint32_t b = cs_div(row, a.by_K), k = row - b * a.c.K;
  const int W = a.c.W, keep = a.keep;
  const int32_t V = (int32_t)a.c.V;
  if (a.finished && a.finished[row]) {   // its one candidate keeps the beam's score; its logits are not read
    if (lane == 0) {
      *stat = BmStat{0.0, 0.0f, base == 0 ? 0.0f : -INF, BM_LOWEST, base == 0 ? 1 : 0};
      if (base == 0) { out_x[0] = 0.0f; out_v[0] = (int32_t)a.c.end_token; }
    }
    return;
  }
  const T* p = (const T*)a.logits + b * a.c.logits_stride[0] + k * a.c.logits_stride[1];
  const uint8_t* mk = MASK ? a.mask + b * a.c.mask_stride[0] + k * a.c.mask_stride[1] : nullptr;
  constexpr int VECS = LANE / N;
  float x[LANE];
  float best = -INF, least = INF;      // (a NaN is passed over)
  float ref = 0.0f;
  double sum = 0.0, sum1 = 0.0;
  const BmPow pow(lane);
  uint32_t raw[VECS][4];
  if (!MASK && base + 64 * LANE <= V) {
#pragma unroll
    for (int j = 0; j < VECS; ++j) __builtin_memcpy(raw[j], p + base + (j * 64 + lane) * N, 16);
    // the sum is formed as the values come in, as if all of them were within [-690, 600] (2^31 terms of exp(600) are far from
    // the end of float64's range); that is seen to below
#pragma unroll
    for (int j = 0; j < VECS; ++j) {
      BmElem<T>::widen(raw[j], x + j * N);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        best = fmaxf(best, x[j * N + e]);
        least = fminf(least, x[j * N + e]);
      }
      if (a.c.normalise) {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          sum = bm_add_exp(sum, (double)x[j * N + e], pow);
          sum1 = bm_add_exp(sum1, (double)x[j * N + e + 1], pow);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  } else {
    // the same where values are not allowed or lie beyond the row's end: -690 in the sum and -inf as a candidate (stretches wholly
    // within the row load without a branch and test the mask alone: 16384 x 4 x 2048 149 us, 192 with one path for both)
    uint8_t m[VECS][N];
    if (MASK && base + 64 * LANE <= V) {
#pragma unroll
      for (int j = 0; j < VECS; ++j) {
        __builtin_memcpy(raw[j], p + base + (j * 64 + lane) * N, 16);
        __builtin_memcpy(m[j], mk + base + (j * 64 + lane) * N, N);
      }
    } else {
#pragma unroll
      for (int j = 0; j < VECS; ++j) {
        const int32_t v0 = base + (j * 64 + lane) * N;
        if (v0 + N <= V) {
          __builtin_memcpy(raw[j], p + v0, 16);
          if (MASK) __builtin_memcpy(m[j], mk + v0, N);
        } else {
          T one[N];
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const int32_t v = v0 + e < V ? v0 + e : V - 1;
            one[e] = p[v];
            if (MASK) m[j][e] = v0 + e < V ? mk[v] : 0;
          }
          __builtin_memcpy(raw[j], one, 16);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < VECS; ++j) {
      BmElem<T>::widen(raw[j], x + j * N);
      float y[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const bool there = MASK ? m[j][e] != 0 : base + (j * 64 + lane) * N + e < V;
        y[e] = there ? x[j * N + e] : -690.0f;
        x[j * N + e] = there ? x[j * N + e] : -INF;
        best = fmaxf(best, x[j * N + e]);
        least = fminf(least, y[e]);
      }
      if (a.c.normalise) {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          sum = bm_add_exp(sum, (double)y[e], pow);
          sum1 = bm_add_exp(sum1, (double)y[e + 1], pow);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  const float top = bm_wave_max(best);
  if (a.c.normalise) {
    if (top < -600.0f || top > 600.0f || __ballot(least < -690.0f)) {
      bool nan = false;
      sum = sum1 = 0.0;
#pragma unroll
      for (int i = 0; i < LANE; ++i) nan = nan || x[i] != x[i];
      if (top > -INF) {
        ref = top;
        // (less than exp(-690) counts as that; of an infinite top every difference is NaN or -inf)
#pragma unroll
        for (int i = 0; i < LANE; ++i) {
          float xi = x[i];
          asm("" : "+v"(xi));   // (else the conversions of both branches are made above them and kept: 64 more registers)
          sum = bm_add_exp(sum, fmax((double)xi - (double)ref, -690.0), pow);
          if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (__ballot(nan) || top == INF) sum = __builtin_nan("");
    }
    sum = bm_wave_sum(sum + sum1);
  }
  // everything from the W-th largest of the lanes' best on is kept
  const uint32_t tk = bm_wave_threshold<16>(best > -INF ? bm_key(best) : 0u, W);
  float t = tk >= bm_key(BM_LOWEST) ? bm_value(tk) : BM_LOWEST;
  const int32_t v_lane = base + lane * N;
  int n = 0;                           // (the same in every lane)
#pragma unroll
  for (int i = 0; i < LANE; ++i) {
    const uint64_t m = __ballot(x[i] >= t);
    if (m) {
      const int c = __popcll(m);
      if (n + c <= keep && x[i] >= t) {
        const uint32_t at = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
        (out_x + n)[at] = x[i];
        (out_v + n)[at] = v_lane + (i / N) * 64 * N + i % N;
      }
      n += c;
    }
  }
  if (n > keep) {
    // too many (W above 32, ascending or equal values): bisect for a bound that W to `keep` of them reach
    uint32_t lo = bm_key(t), hi = bm_key(top) + 1;   // W or more reach lo, none hi
    int c = n;
    while (c > keep && hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      const float f = bm_value(mid);
      int reach = 0;
#pragma unroll
      for (int i = 0; i < LANE; ++i) reach += __popcll(__ballot(x[i] >= f));
      if (reach < W) hi = mid;
      else { lo = mid; c = reach; }
    }
    t = bm_value(lo);
    const bool equal = c > keep;       // none found: lo is the W-th largest value, and others equal it
    n = 0;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // other lanes stored to these places above
#pragma unroll
    for (int i = 0; i < LANE; ++i) {
      const bool take = equal ? x[i] > t : x[i] >= t;
      const uint64_t m = __ballot(take);
      const uint32_t at = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
      if (take) {
        (out_x + n)[at] = x[i];
        (out_v + n)[at] = v_lane + (i / N) * 64 * N + i % N;
      }
      n += __popcll(m);
    }
    if (equal) {   // of those equal to it the first ones
#pragma unroll
      for (int j = 0; j < LANE / N; ++j) {
        int mine = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) mine += x[j * N + e] == t;
        int incl = mine;
        for (int o = 1; o < 64; o <<= 1) {
          const int other = __shfl_up(incl, o);
          if (lane >= o) incl += other;
        }
        int at = n + incl - mine;
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (x[j * N + e] == t) {
            if (at < W) { out_x[at] = t; out_v[at] = v_lane + j * 64 * N + e; }
            ++at;
          }
        n += __shfl(incl, 63);
      }
      n = n < W ? n : W;
      float down = -INF;
#pragma unroll
      for (int i = 0; i < LANE; ++i) {
        float xi = x[i];
        asm("" : "+v"(xi));   // (else the comparisons above are kept for these, 32 pairs of registers)
        down = fmaxf(down, xi < t ? xi : -INF);
      }
      down = bm_wave_max(down);
      if (lane == 0) {
        out_x[n] = down;
        *stat = BmStat{sum, ref, top, __builtin_nanf(""), n};
      }
      return;
    }
  }
  if (lane == 0) *stat = BmStat{sum, ref, top, t, n};
}

// (float32 without a mask fits 6 wavefronts on a SIMD when asked to, 2 % faster; masked kernels spill and lose a quarter)
template <typename T, bool MASK, int LANE>
__global__ void __launch_bounds__(256, LANE == 32 && !MASK && BmElem<T>::N == 4 ? 6 : 1) cs_beam_scan_kernel(const BmArgs a) {
  const uint32_t item = cs_block() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= a.items) return;
  const uint32_t row = cs_div(item, a.by_stretches);
  const int64_t at = (int64_t)item * a.keep;
  bm_scan<T, MASK, LANE>(a, row, item - row * a.stretches, a.stat + item, a.item_x + at, a.item_v + at);
}

// One workgroup per example; bound by its chain of dependent loads and barriers: 6.8 us for 4 beams of 32 stretches, 15 for 16 of
// 64, 10 for 4096 examples of 5 stretches (W = 64: 46).  Lists that have to be completed cost the most where every beam's score swallows
// its logits (all at -1e30): 4096 x 10200 in 75 us instead of 44, 64 x 16 x 131072 in 1.7 ms instead of 0.1.
__device__ __forceinline__ void bm_join(int64_t b, BmStat* stat, float* item_x, int32_t* item_v, char* lds, int cap) {
  const BmArgs& a = bm_args();
  double* s_lse = (double*)lds;                                     // [K]
  double* s_before = s_lse + a.c.K;                                 // [K] scores
  uint64_t* s_key = (uint64_t*)(s_before + a.c.K);                  // [cap] scores of candidates, as ordered bits
  int64_t* s_at = (int64_t*)(s_key + cap);                          // [cap] k << 32 | v
  __shared__ uint64_t s_wave[BM_JOIN / 64];
  __shared__ int64_t s_wave_at[BM_JOIN / 64];
  int* s_open = (int*)(s_at + cap);                                 // [threads, at least 192] stretches to go through
  __shared__ int s_n, s_left, s_left_out, s_greater;
  __shared__ uint64_t s_edge;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int threads = blockDim.x, waves = threads >> 6;
  const int K = a.c.K, W = a.c.W, C = a.stretches, keep = a.keep;
  const int32_t total = K * C;         // (at most 2^31 / keep, checked on the host)
  constexpr double INF = __builtin_inf();
  // (asked for before the normalisers are formed)
  const float top0 = tid < total ? stat[tid].top : -__builtin_inff();
  const int n0 = tid < total ? stat[tid].n : 0;
  const int n_first = total <= 64 && lane < total ? stat[lane].n : 0;
  const BmPow pow(lane);
  if (tid == 0) { s_n = 0; s_left = 0; s_left_out = 0; }
  // the lanes of a beam: a power of two
  int g = 1;
  while (g < C && g < 64) g *= 2;
  const int per = 64 / g, sub = lane & (g - 1);
  for (int k0 = wave * per; k0 < K; k0 += waves * per) {
    const int k = k0 + lane / g;
    const bool mine = k < K;
    const int64_t row = b * K + (mine ? k : K - 1);
    double before = 0.0, lse = 0.0;
    if (a.scores) before = a.c.scores_type == CS_TYPE_F64 ? ((const double*)a.scores)[row] : (double)((const float*)a.scores)[row];
    const bool formed = mine && a.c.normalise && !(a.finished && a.finished[row]);
    if (__ballot(formed)) {
      const BmStat* st = stat + k * C;
      // Lanes join their stretches, then each other: those of reference 0 (the rule) and, apart, the others.
      float top = -__builtin_inff();               // of the former
      double sum = 0.0, ref = -INF, far = 0.0;     // far: of the latter, relative to ref
      for (int c = sub; formed && c < C; c += g) {
        const BmStat s = st[c];
        if (s.sum != s.sum) sum = s.sum;             // (NaN stays)
        if (!(s.top > -__builtin_inff())) continue;  // nothing allowed there
        if (s.ref == 0.0f) {
          top = fmaxf(top, s.top);
          sum += s.sum;
        } else {
          const double m = fmax(ref, (double)s.ref);
          far = far * exp(ref - m) + s.sum * exp((double)s.ref - m);
          ref = m;
        }
      }
      if (g == 64) {
        top = bm_wave_max(top);
        sum = bm_wave_sum(sum);
      } else {
        for (int o = g >> 1; o; o >>= 1) {
          top = fmaxf(top, __shfl_xor(top, o));
          sum += __shfl_xor(sum, o);
        }
      }
      double m = (double)top;
      if (__ballot(ref > -INF)) {
        double all = ref;
        for (int o = g >> 1; o; o >>= 1) all = fmax(all, __shfl_xor(all, o));
        far = ref > -INF ? far * exp(ref - all) : far;
        for (int o = g >> 1; o; o >>= 1) far += __shfl_xor(far, o);
        m = fmax(m, all);
        far = all > -INF ? far * exp(all - m) : far;
      }
      // The sum relative to the largest logit, that logit's own part being one exactly: a beam left with one value has a
      // normaliser of just its logit, and of a beam that is all but certain the rest counts, not the roundings of the whole.
      const double e = bm_add_exp(0.0, m, pow);      // (all lanes have to be there)
      if (m == (double)top) sum = 1.0 + (sum - e) / e;
      else if (top > -__builtin_inff()) sum *= exp(-m);
      lse = formed ? m + log(sum + far) : 0.0;       // (+inf, NaN or nothing allowed: NaN or -inf, with no candidate left to count)
    }
    if (mine && sub == 0) { s_lse[k] = lse; s_before[k] = before; }
  }
  __syncthreads();
  auto key_of = [&](float x, int g) {   // (in this order: where x is the whole normaliser, the score stays what it was)
    const uint32_t k = cs_div(g, a.by_stretches);
    return bm_key64(s_before[k] + ((double)x - s_lse[k]));
  };
  // The best score that stretch g may have left out, 0 for none.  Within a beam it is no better than W kept ones, and it counts only
  // where it is no worse than the worst of these: where one score has logits on both sides of the bound.
  auto left_out = [&](int g) -> uint64_t {
    const float cut = stat[g].cut;
    if (cut == BM_LOWEST) return 0;
    if (cut == cut) {   // (the float32 before it; both zeros are one)
      const uint64_t at = key_of(cut, g);
      return key_of(cut == 0.0f ? -1.401298464e-45f : bm_value(bm_key(cut) - 1), g) == at ? at : 0;
    }
    const float* x = item_x + (int64_t)g * keep;        // (the larger ones come first)
    const int n = stat[g].n;
    const float last = x[n - 1];
    const uint64_t at = key_of(last, g);
    bool one = x[n] > -__builtin_inff() && key_of(x[n], g) == at;
    for (int r = 0; !one && x[r] > last; ++r) one = key_of(x[r], g) == at;
    return one ? at : 0;
  };
  // a bound from below; none where there are few candidates
  uint64_t t = 1;
  if (total > 64 || bm_wave_sum((double)n_first) > 2 * W + 64) {
    // the W-th largest score, as far as its leading 32 bits say, among the lanes' best of a wavefront: of the stretches' largest
    // logits or, where these are few, of all kept ones
    uint32_t best = 0;
    if (total >= 4 * W) {
      for (int g = tid; g < total; g += threads) {
        const float x = g == tid ? top0 : stat[g].top;
        const uint32_t key = x > -__builtin_inff() ? (uint32_t)(key_of(x, g) >> 32) : 0u;
        best = key > best ? key : best;
      }
    } else {
      for (uint32_t i = tid; i < (uint32_t)(total * keep); i += threads) {   // (the product is below 2^31, the sum may pass it)
        const int g = cs_div(i, a.by_keep);
        if ((int)i - g * keep < stat[g].n) {
          const uint32_t key = (uint32_t)(key_of(item_x[i], g) >> 32);
          best = key > best ? key : best;
        }
      }
    }
    const uint32_t t_wave = bm_wave_threshold<32>(best, W);
    if (lane == 0) s_wave[wave] = t_wave;
    __syncthreads();
    uint32_t t32 = 1;
    for (int w = 0; w < waves; ++w) t32 = s_wave[w] > t32 ? (uint32_t)s_wave[w] : t32;
    // where many of the lanes' best are left, the W-th largest of these (4 us; ranking the hundreds of candidates that are above
    // the first bound took 10)
    const uint64_t reach = __ballot(best >= t32);
    if (waves > 1) {
      if (lane == 0) atomicAdd(&s_left, __popcll(reach));
      __syncthreads();
      const int left = s_left;
      if (left > 4 * W) {
        uint32_t* s_best = (uint32_t*)s_key;           // [threads] (threads <= 2 cap)
        if (best >= t32) s_best[atomicAdd(&s_n, 1)] = best;
        __syncthreads();
        if (tid == 0) { s_n = 0; s_wave[0] = t32; }
        __syncthreads();
        if (tid < left) {
          const uint32_t mine = s_best[tid];
          int before = 0;
#pragma unroll 8
          for (int j = 0; j < left; ++j) before += s_best[j] > mine || (s_best[j] == mine && j < tid);
          if (before == W - 1) s_wave[0] = mine;
        }
        __syncthreads();
        t32 = (uint32_t)s_wave[0];
      }
    }
    t = t32 > 1 ? (uint64_t)t32 << 32 : 1;
  }
  uint64_t below = 0;                  // the best score that this thread's stretches may have left out
  // stretches whose largest logit reaches the bound are gone through by 16 lanes each
  for (int g0 = 0; g0 < total; g0 += threads) {
    __syncthreads();
    if (tid == 0) s_left = 0;
    __syncthreads();
    const int g = g0 + tid;
    if (g < total) {
      const float x = g0 == 0 ? top0 : stat[g].top;
      if (x > -__builtin_inff() && key_of(x, g) >= t) {
        s_open[atomicAdd(&s_left, 1)] = g;
        const uint64_t u = left_out(g);
        if (u >= t) { below = u > below ? u : below; s_left_out = 1; }
      }
    }
    __syncthreads();
    const int open = s_left;
    for (int o = tid >> 4; o < open; o += threads >> 4) {
      const int h = s_open[o], n = g0 == 0 && h == tid ? n0 : stat[h].n;
      for (int r = tid & 15; r < n; r += 16) {
        const int64_t i = (int64_t)h * keep + r;
        const uint64_t key = key_of(item_x[i], h);
        if (key < t) continue;
        const int at = atomicAdd(&s_n, 1);   // (places in any order: the ranks below depend on the entries alone)
        if (at < cap) { s_key[at] = key; s_at[at] = (int64_t)cs_div(h, a.by_stretches) << 32 | item_v[i]; }
      }
    }
  }
  __syncthreads();
  auto put = [&](int w, uint64_t key, int64_t at) {
    const int64_t o = b * W + w;
    const double s = key ? bm_value64(key) : -INF;
    if (a.c.scores_type == CS_TYPE_F64) ((double*)a.out_scores)[o] = s;
    else ((float*)a.out_scores)[o] = (float)s;
    a.parents[o] = key ? at >> 32 : (w < K ? w : K - 1);
    a.tokens[o] = key ? at & 0xffffffff : -1;
  };
  const int n = s_n;
  uint64_t edge = 0;                   // the W-th best score, and how many results are better
  int greater = 0;
  if (n <= cap) {
    // ranks by counting: each candidate against all.  Where there are many (W above 32), those from a bound on that W to 32
    // more reach, bisected
    int m = n;
    if (n > W + 96) {
      uint64_t most = 0;
      for (int i = tid; i < n; i += threads) most = s_key[i] > most ? s_key[i] : most;
      for (int o = 32; o; o >>= 1) {
        const uint64_t u = __shfl_xor((unsigned long long)most, o);
        most = u > most ? u : most;
      }
      __syncthreads();
      if (lane == 0) s_wave[wave] = most;
      __syncthreads();
      for (int w = 0; w < waves; ++w) most = s_wave[w] > most ? s_wave[w] : most;
      uint64_t lo = t, hi = most + 1;              // W or more reach lo, none hi
      int left = n;
      while (left > W + 32 && hi - lo > 1) {
        const uint64_t mid = lo + (hi - lo) / 2;
        __syncthreads();
        if (tid == 0) s_left = 0;
        __syncthreads();
        int reach = 0;
        for (int i = tid; i < n; i += threads) reach += s_key[i] >= mid;
        for (int o = 32; o; o >>= 1) reach += __shfl_xor(reach, o);
        if (lane == 0) atomicAdd(&s_left, reach);
        __syncthreads();
        if (s_left < W) hi = mid;
        else { lo = mid; left = s_left; }
      }
      if (left <= W + 32) {                        // (else that many are equal: all stay)
        __syncthreads();
        if (tid == 0) s_left = 0;
        __syncthreads();
        for (int i = tid; i < n; i += threads)
          if (s_key[i] >= lo) s_open[atomicAdd(&s_left, 1)] = i;
        __syncthreads();
        // they move to the front: two at most of a thread
        const int i0 = tid < left ? s_open[tid] : 0, i1 = tid + 64 < left && tid < 64 ? s_open[tid + 64] : 0;
        const uint64_t k0 = s_key[i0], k1 = s_key[i1];
        const int64_t at0 = s_at[i0], at1 = s_at[i1];
        __syncthreads();
        if (tid < left && tid < 64) { s_key[tid] = k0; s_at[tid] = at0; }
        if (tid + 64 < left && tid < 64) { s_key[tid + 64] = k1; s_at[tid + 64] = at1; }
        __syncthreads();
        m = left;
      }
    }
    for (int i = tid; i < m; i += threads) {
      const uint64_t key = s_key[i];
      const int64_t at = s_at[i];
      int before = 0, equal = 0;
#pragma unroll 8
      for (int j = 0; j < m; ++j) {
        const uint64_t other = s_key[j];
        before += other > key;
        equal += other == key;
      }
      const int more = before;
      if (equal > 1 && before < W)
        for (int j = 0; j < m; ++j) before += s_key[j] == key && s_at[j] < at;
      if (before < W) put(before, key, at);
      if (before == W - 1) { s_edge = key; s_greater = more; }
    }
    for (int w = n + tid; w < W; w += threads) put(w, 0, 0);
    if (n < W || !s_left_out) return;
    __syncthreads();
    edge = s_edge;
    if (below >= edge) s_left_out = 2;
    __syncthreads();
    if (s_left_out != 2) return;
    greater = s_greater;
  }
  // many equal scores: the results one by one, each the best of what comes after the one before
  for (;;) {
    if (edge) {
      // Stretches that may have left out some of the W-th best score get lists that are whole: of what they kept the better ones, and
      // then the first values of that score.  A wavefront per stretch.
      auto ahead = [](uint64_t m) { return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0)); };
      const BmArgs& args = bm_args();
      const int want = W - greater;                // (in all; with the better ones of a stretch no more than W)
      for (int g = wave; g < total; g += waves) {
        if (!(stat[g].top > -__builtin_inff()) || left_out(g) < edge) continue;
        const int n = stat[g].n;
        float* gx = item_x + (int64_t)g * keep;
        int32_t* gv = item_v + (int64_t)g * keep;
        int c = 0;
        for (int r0 = 0; r0 < n; r0 += 64) {       // (to places that have been read: the stores wait for the loads)
          const bool there = r0 + lane < n;
          const float x = there ? gx[r0 + lane] : 0.0f;
          const int32_t v = there ? gv[r0 + lane] : 0;
          const bool better = there && key_of(x, g) > edge;
          const uint64_t m = __ballot(better);
          if (better) { gx[c + ahead(m)] = x; gv[c + ahead(m)] = v; }
          c += __popcll(m);
        }
        const int k = (int)cs_div(g, a.by_stretches);
        const int64_t at = b * args.c.logits_stride[0] + k * args.c.logits_stride[1], mask_at = b * args.c.mask_stride[0] + k * args.c.mask_stride[1];
        const int64_t v1 = (int64_t)(g - k * C + 1) * args.len, end = v1 < args.c.V ? v1 : args.c.V;
        int found = 0;
        for (int64_t v0 = v1 - args.len; v0 < end && found < want; v0 += 64) {
          const int64_t v = v0 + lane;
          float x = -__builtin_inff();
          if (v < end && !(args.mask && !args.mask[mask_at + v])) {
            if (args.c.logits_type == CS_TYPE_F32) x = ((const float*)args.logits)[at + v];
            else if (args.c.logits_type == CS_TYPE_BF16) x = __uint_as_float((uint32_t)((const uint16_t*)args.logits)[at + v] << 16);
            else x = (float)((const _Float16*)args.logits)[at + v];
          }
          const bool mine = x > -__builtin_inff() && key_of(x, g) == edge;
          const uint64_t m = __ballot(mine);
          const int place = c + found + ahead(m);
          if (mine && place < c + want) { gx[place] = x; gv[place] = (int32_t)v; }
          found += __popcll(m);
        }
        if (lane == 0) stat[g].n = c + (found < want ? found : want);
      }
      __syncthreads();
    }
    uint64_t last = ~0ull;
    int64_t last_at = -1;
    for (int w = 0; w < W; ++w) {
      uint64_t key = 0;
      int64_t at = 0;
      for (uint32_t i = tid; i < (uint32_t)(total * keep); i += threads) {
        const int g = cs_div(i, a.by_keep);
        if ((int)i - g * keep >= stat[g].n) continue;
        const uint64_t u = key_of(item_x[i], g);
        const int64_t f = (int64_t)cs_div(g, a.by_stretches) << 32 | item_v[i];
        if ((u < last || (u == last && f > last_at)) && (u > key || (u == key && key && f < at))) { key = u; at = f; }
      }
      for (int o = 32; o; o >>= 1) {
        const uint64_t u = __shfl_xor((unsigned long long)key, o);
        const int64_t f = __shfl_xor((long long)at, o);
        if (u > key || (u == key && f < at)) { key = u; at = f; }
      }
      __syncthreads();
      if (lane == 0) { s_wave[wave] = key; s_wave_at[wave] = at; }
      __syncthreads();
      key = s_wave[0]; at = s_wave_at[0];
      for (int v = 1; v < waves; ++v)
        if (s_wave[v] > key || (s_wave[v] == key && s_wave_at[v] < at)) { key = s_wave[v]; at = s_wave_at[v]; }
      if (tid == 0) put(w, key, at);
      if (key != last) greater = w;
      last = key;
      last_at = key ? at : INT64_MAX;
    }
    if (edge || !last) return;
    edge = last;
    if (below >= edge) s_left_out = 2;
    __syncthreads();
    if (s_left_out != 2) return;
  }
}

__global__ void __launch_bounds__(BM_JOIN) cs_beam_join_kernel(const BmArgs a, int cap) {
  extern __shared__ __align__(16) char lds[];
  const int64_t b = cs_block(), total = (int64_t)a.c.K * a.stretches;
  if (b >= a.c.B) return;
  bm_join(b, a.stat + b * total, a.item_x + b * total * a.keep, a.item_v + b * total * a.keep, lds, cap);
}

// Both in one launch, where an example has few stretches: a wavefront each, which leave what they keep in LDS.  Saves a launch (512 x
// 4 x 10: 12 us per call, not 15) and the way through memory (16384 x 4 x 2048: 132, not 165).  Where several stretches of 2048 make
// a beam it loses, since a workgroup loads nothing while it joins (4096 x 10200: 67, not 47): there the two launches stay.
template <typename T, bool MASK, int LANE>
__global__ void __launch_bounds__(BM_ONE * 64) cs_beam_one_kernel(const BmArgs a, int cap) {
  extern __shared__ __align__(16) char lds[];
  const int64_t b = cs_block();
  if (b >= a.c.B) return;
  const int total = a.c.K * a.stretches, keep = a.keep;
  BmStat* stat = (BmStat*)lds;
  float* item_x = (float*)(stat + total);
  int32_t* item_v = (int32_t*)(item_x + total * keep);
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), k = cs_div(w, a.by_stretches);
  bm_scan<T, MASK, LANE>(a, (uint32_t)b * a.c.K + k, w - k * a.stretches, stat + w, item_x + w * keep, item_v + w * keep);
  __syncthreads();
  bm_join(b, stat, item_x, item_v, lds + total * (sizeof(BmStat) + keep * 8), cap);
}

// values per lane of a stretch: 32 where that fills the chip (6 wavefronts on each of its 1024 SIMDs), else, or where fewer hold
// all values, 16 or 8
int lane_values(const cs_beam_cfg& c) {
  int lane = 32;
  while (lane > 8 && (c.V <= 32 * lane || (int64_t)c.B * c.K * ((c.V + 64 * lane - 1) / (64 * lane)) < 6144)) lane /= 2;
  return lane;
}
int32_t stretches_of(const cs_beam_cfg& c) {
  const int64_t len = 64 * lane_values(c);
  return (int32_t)((c.V + len - 1) / len);
}
// places for the logits kept of a stretch: what lies above the W-th largest of its lanes' best is a few more than W for
// W <= 32; for more, nearly all lanes count, their best tell little, and a better bound is bisected
int32_t keep_of(const cs_beam_cfg& c) { return c.W <= 32 ? 2 * c.W + 32 : 96; }

// the scan alone or, given its threads, the kernel that joins as well
template <typename T, bool MASK, int LANE>
void launch_stretches(const BmArgs& a, int threads, int lds, int cap, hipStream_t st) {
  if (threads) hipLaunchKernelGGL((cs_beam_one_kernel<T, MASK, LANE>), cs_grid(a.c.B), dim3(threads), lds, st, a, cap);
  else hipLaunchKernelGGL((cs_beam_scan_kernel<T, MASK, LANE>), cs_grid(((int64_t)a.items + 3) / 4), dim3(256), 0, st, a);
}
template <typename T>
void launch_scan(const BmArgs& a, int threads, int lds, int cap, hipStream_t st) {
  switch (lane_values(a.c)) {
#define CS_SCAN(L_)                                                                \
    case L_:                                                                       \
      if (a.mask) launch_stretches<T, true, L_>(a, threads, lds, cap, st);         \
      else launch_stretches<T, false, L_>(a, threads, lds, cap, st);               \
      break;
    CS_SCAN(8) CS_SCAN(16) CS_SCAN(32)
#undef CS_SCAN
  }
}

int check_beam(const cs_beam_cfg* c) {
  CS_REQUIRE(c, "null argument");
  CS_REQUIRE(c->B >= 0 && c->K >= 1 && c->K <= BM_MAXK, "1 .. 2048 beams");
  CS_REQUIRE(c->V >= 1 && c->V <= (int64_t)INT32_MAX - 65536, "bad number of values");
  CS_REQUIRE(c->W >= 1 && c->W <= BM_MAXW, "width must be 1 .. 64");
  CS_REQUIRE(c->logits_type == CS_TYPE_F32 || c->logits_type == CS_TYPE_BF16 || c->logits_type == CS_TYPE_F16,
             "logits are float32, bfloat16 or float16");
  CS_REQUIRE(c->scores_type == CS_TYPE_F32 || c->scores_type == CS_TYPE_F64, "scores are float32 or float64");
  CS_REQUIRE((int64_t)c->K * stretches_of(*c) <= INT32_MAX / keep_of(*c) && (int64_t)c->B * c->K <= INT32_MAX / stretches_of(*c),
             "too many logits for one call");
  return CS_OK;
}

}  // namespace

extern "C" int64_t cs_beam_select_workspace(const cs_beam_cfg* c) {
  if (check_beam(c)) return -1;
  return (int64_t)c->B * c->K * stretches_of(*c) * (int64_t)(sizeof(BmStat) + keep_of(*c) * 8);
}

extern "C" int cs_beam_select(const cs_beam_cfg* c, const void* scores, const void* logits, const uint8_t* mask,
                              const uint8_t* finished, void* out_scores, int64_t* parents, int64_t* tokens, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  if (int rc = check_beam(c)) return rc;
  CS_REQUIRE(!finished || (c->end_token >= 0 && c->end_token < c->V), "end token outside the values");
  if (c->B == 0) return CS_OK;
  CS_REQUIRE(logits && out_scores && parents && tokens && workspace, "null argument");
  CS_REQUIRE(workspace_bytes >= cs_beam_select_workspace(c), "workspace too small");
  CS_REQUIRE(((uintptr_t)workspace & 7) == 0, "workspace must be 8-byte aligned");
  BmArgs a;
  a.c = *c;
  a.scores = scores; a.logits = logits; a.mask = mask; a.finished = finished;
  a.stretches = stretches_of(*c);
  a.keep = keep_of(*c);
  a.len = 64 * lane_values(*c);
  const int64_t items = (int64_t)c->B * c->K * a.stretches;
  a.stat = (BmStat*)workspace;
  a.item_x = (float*)(a.stat + items);
  a.item_v = (int32_t*)(a.item_x + items * a.keep);
  a.out_scores = out_scores; a.parents = parents; a.tokens = tokens;
  hipStream_t st = (hipStream_t)stream;
  a.items = (uint32_t)items;
  a.by_stretches = cs_div_by(a.stretches);
  a.by_K = cs_div_by(c->K);
  a.by_keep = cs_div_by(a.keep);
  const int64_t total = (int64_t)c->K * a.stretches;
  const bool one = total <= BM_ONE && (a.stretches == 1 || lane_values(*c) < 32);
  // a thread per stretch, those of a beam in one wavefront, as far as that goes
  int lanes = 1;
  while (lanes < a.stretches && lanes < 64) lanes *= 2;
  int64_t waves = ((total > c->K * lanes ? total : c->K * lanes) + 63) / 64;
  // (16 lanes go through what is kept of a stretch: up to 4 wavefronts while the chip has room for them.  1024 x 4 x 8000, 16
  // stretches: 36 us with 4, 45 with 1; 4096 x 1 x 32000, 16 as well: 122 with 4, 111 with 1)
  int64_t few = total / 4 < 4 ? total / 4 : 4;
  few = few < 4096 / c->B ? few : 4096 / c->B;
  waves = few > waves ? few : waves;
  // (and for wide searches a thread for every 8 of some W candidates per stretch, so that the W-th largest of the threads' best
  // is a good bound)
  const int64_t wide = (total * c->W + 511) / 512;
  waves = c->W > 32 && wide > waves ? wide : waves;
  waves = one ? total : waves < BM_JOIN / 64 ? waves : BM_JOIN / 64;
  const int threads = 64 * (int)waves;
  // places for what reaches the joined bound
  const int least = threads == 64 ? 128 : 1024, most = c->K > 1024 ? 1024 : 2048;   // (64 KB of LDS in all)
  int cap = c->W * 32;
  cap = cap > most ? most : cap < least ? least : cap;
  if (total <= 64 && cap > total * a.keep) cap = (int)total * a.keep;
  const int lds = c->K * 16 + cap * 16 + (threads < 192 ? 192 : threads) * 4;
  const int lds_one = lds + (int)total * (int)(sizeof(BmStat) + a.keep * 8);
  if (c->logits_type == CS_TYPE_F32) launch_scan<float>(a, one ? threads : 0, lds_one, cap, st);
  else if (c->logits_type == CS_TYPE_BF16) launch_scan<BmBf16>(a, one ? threads : 0, lds_one, cap, st);
  else launch_scan<_Float16>(a, one ? threads : 0, lds_one, cap, st);
  CS_HIP(hipGetLastError());
  if (!one) {
    hipLaunchKernelGGL(cs_beam_join_kernel, cs_grid(c->B), dim3(threads), (size_t)lds, st, a, cap);
    CS_HIP(hipGetLastError());
  }
  return CS_OK;
}

// ---- states that follow their parents -----------------------------------------------------------------------------
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct BmMoveArgs {
  const char* src;
  char* dst;
  const int64_t* parents;
  int64_t outer, B, cols;              // cols: pieces of a row
  int64_t full;                        // the first ones are of the wider type, at any address
  int64_t ss[3], ds[3];                // bytes between outer / example / chain
  int32_t K, W;
  int64_t outer_step;                  // a thread serves every outer_step-th outer index
  int32_t small;                       // all pieces of an outer index are less than 2^32
  CsDiv by_cols, by_W;
};

__device__ __forceinline__ int64_t bm_over(const BmMoveArgs& a, int64_t n, const CsDiv& by, int64_t d) {
  return a.small ? (int64_t)cs_div((uint32_t)n, by) : n / d;
}
template <typename V> __device__ __forceinline__ V bm_get(const char* p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}
template <typename V> __device__ __forceinline__ void bm_put(char* p, V v) { __builtin_memcpy(p, &v, sizeof(V)); }

template <typename V>
__device__ __forceinline__ void bm_gather(const BmMoveArgs& a, const char* s, char* d) {
  for (int64_t o = blockIdx.z; o < a.outer; o += a.outer_step) bm_put(d + o * a.ds[0], bm_get<V>(s + o * a.ss[0]));
}
// out of place: a thread per piece of a destination row, over its outer indices
template <typename FULL, typename VEC>
__global__ void __launch_bounds__(256) cs_beam_gather_kernel(const BmMoveArgs a) {
  const int64_t i = (int64_t)cs_block() * 256 + threadIdx.x;
  if (i >= a.B * a.W * a.cols) return;
  const int64_t bw = bm_over(a, i, a.by_cols, a.cols), col = i - bw * a.cols;
  const int64_t p = a.parents[bw];
  if (p < 0 || p >= a.K) return;
  const int64_t b = bm_over(a, bw, a.by_W, a.W), w = bw - b * a.W;
  const char* s = a.src + b * a.ss[1] + p * a.ss[2];
  char* d = a.dst + b * a.ds[1] + w * a.ds[2];
  if (sizeof(FULL) == sizeof(VEC) || col < a.full) {
    bm_gather<FULL>(a, s + col * sizeof(FULL), d + col * sizeof(FULL));
  } else {
    const int64_t at = a.full * sizeof(FULL) + (col - a.full) * sizeof(VEC);
    bm_gather<VEC>(a, s + at, d + at);
  }
}

// In place a thread owns one piece of all K rows of an example, so it reads every row it needs before it writes any; rows that
// keep their place are neither read nor written.
template <typename V, int KMAX>
__device__ __forceinline__ void bm_move_few(const BmMoveArgs& a, char* d, const int (&parent)[KMAX]) {
  for (int64_t o = blockIdx.z; o < a.outer; o += a.outer_step) {
    V v[KMAX];
#pragma unroll
    for (int k = 0; k < KMAX; ++k)
      if (parent[k] >= 0) v[k] = bm_get<V>(d + o * a.ds[0] + parent[k] * a.ds[2]);
#pragma unroll
    for (int k = 0; k < KMAX; ++k)
      if (parent[k] >= 0) bm_put(d + o * a.ds[0] + k * a.ds[2], v[k]);
  }
}
template <typename V, int KMAX, typename MASK>
__device__ __forceinline__ void bm_move(const BmMoveArgs& a, char* d, MASK moved, const uint8_t* parent) {
  auto first = [](MASK m) { return sizeof(MASK) == 8 ? __builtin_ctzll(m) : __builtin_ctz((uint32_t)m); };
  for (int64_t o = blockIdx.z; o < a.outer; o += a.outer_step) {
    char* at = d + o * a.ds[0];
    V v[KMAX];
    MASK rest = moved;
#pragma unroll
    for (int j = 0; j < KMAX; ++j)
      if (rest) {
        v[j] = bm_get<V>(at + parent[first(rest)] * a.ds[2]);
        rest &= rest - 1;
      }
    rest = moved;
#pragma unroll
    for (int j = 0; j < KMAX; ++j)
      if (rest) {
        bm_put(at + first(rest) * a.ds[2], v[j]);
        rest &= rest - 1;
      }
  }
}

// Up to 4 chains: each thread reads its example's parents.  Bound by memory in whole lines of 128 bytes: half of
// 4 chains moved, 211 MB of moved bytes read and written, takes 50 us in rows of 128 bytes (4.2 TB/s), 44 in rows of 1 KB and
// 80 in rows of 172 bytes, whose ends share lines with rows that stay.  (There, 16 bytes a lane measured 81, scalar parents
// with several columns a lane 86, streaming stores and loads 93 and 107.)
template <typename FULL, typename VEC>
__global__ void __launch_bounds__(256) cs_beam_inplace_few_kernel(const BmMoveArgs a) {
  const int64_t i = (int64_t)cs_block() * 256 + threadIdx.x;
  if (i >= a.B * a.cols) return;
  const int64_t b = bm_over(a, i, a.by_cols, a.cols), col = i - b * a.cols;
  int parent[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t p = k < a.K ? a.parents[b * a.K + k] : -1;
    parent[k] = p < 0 || p >= a.K || p == k ? -1 : (int)p;
  }
  char* d = a.dst + b * a.ds[1];
  if (sizeof(FULL) == sizeof(VEC) || col < a.full) bm_move_few<FULL>(a, d + col * sizeof(FULL), parent);
  else bm_move_few<VEC>(a, d + a.full * sizeof(FULL) + (col - a.full) * sizeof(VEC), parent);
}

// More: the workgroup's parents lie in LDS and a thread goes through the bits of the rows that move alone (2 of 10 rows of 818 bytes:
// 11 us; with a test per chain and the parents in registers 23).
template <typename FULL, typename VEC, int KMAX>
__global__ void __launch_bounds__(256) cs_beam_inplace_kernel(const BmMoveArgs a) {
  using MASK = typename std::conditional<(KMAX > 32), unsigned long long, unsigned>::type;
  constexpr int EXAMPLES = 257;        // of a workgroup, at most
  __shared__ MASK s_moved[EXAMPLES];
  __shared__ uint8_t s_parent[EXAMPLES * KMAX];
  const int tid = threadIdx.x;
  const int64_t pieces = a.B * a.cols, i0 = (int64_t)cs_block() * 256;
  if (i0 >= pieces) return;
  const int64_t i = i0 + tid < pieces ? i0 + tid : pieces - 1, last = i0 + 255 < pieces ? i0 + 255 : pieces - 1;
  const int64_t b0 = bm_over(a, i0, a.by_cols, a.cols), b = bm_over(a, i, a.by_cols, a.cols);
  const int examples = (int)(bm_over(a, last, a.by_cols, a.cols) - b0) + 1;
  for (int e = tid; e < examples; e += 256) s_moved[e] = 0;
  __syncthreads();
  for (int e = tid; e < examples * a.K; e += 256) {
    const int x = (int)cs_div((uint32_t)e, a.by_W), k = e - x * a.K;     // (W = K)
    const int64_t p = a.parents[b0 * a.K + e];
    if (p >= 0 && p < a.K && p != k) {
      s_parent[x * KMAX + k] = (uint8_t)p;
      atomicOr(&s_moved[x], (MASK)1 << k);
    }
  }
  __syncthreads();
  if (i0 + tid >= pieces) return;
  const MASK moved = s_moved[b - b0];
  const uint8_t* parent = s_parent + (b - b0) * KMAX;
  const int64_t col = i - b * a.cols;
  char* d = a.dst + b * a.ds[1];
  if (sizeof(FULL) == sizeof(VEC) || col < a.full) bm_move<FULL, KMAX>(a, d + col * sizeof(FULL), moved, parent);
  else bm_move<VEC, KMAX>(a, d + a.full * sizeof(FULL) + (col - a.full) * sizeof(VEC), moved, parent);
}

// The bytes of a piece where starts and ends of all rows are multiples of `unit` bytes: the unit, or 16 (8, 4 where a thread holds more
// than 16, 32 of them) at any address and what is left of a row in units.  The latter pays where a row has many units: 785 bytes in 5
// chains, 2 moved: 81 us, not 191; 1700 bytes, out of place: 44, not 57; but 172 bytes: 34, not 30.
int piece_of(int unit, int64_t row_bytes, bool in_place, int K) {
  const int widest = !in_place || K <= 16 ? 16 : K <= 32 ? 8 : 4;
  return unit <= 2 || (unit == 4 && row_bytes >= 256) || unit > widest ? widest : unit;
}
template <typename FULL, typename VEC>
void launch_pieces(const BmMoveArgs& a, bool in_place, dim3 grid, hipStream_t st) {
  if (!in_place) hipLaunchKernelGGL((cs_beam_gather_kernel<FULL, VEC>), grid, dim3(256), 0, st, a);
  else if (a.K <= 4) hipLaunchKernelGGL((cs_beam_inplace_few_kernel<FULL, VEC>), grid, dim3(256), 0, st, a);
  else if (a.K <= 8) hipLaunchKernelGGL((cs_beam_inplace_kernel<FULL, VEC, 8>), grid, dim3(256), 0, st, a);
  else if (a.K <= 16) hipLaunchKernelGGL((cs_beam_inplace_kernel<FULL, VEC, 16>), grid, dim3(256), 0, st, a);
  else if constexpr (sizeof(FULL) == 8) hipLaunchKernelGGL((cs_beam_inplace_kernel<FULL, VEC, 32>), grid, dim3(256), 0, st, a);
  else if constexpr (sizeof(FULL) == 4) hipLaunchKernelGGL((cs_beam_inplace_kernel<FULL, VEC, 64>), grid, dim3(256), 0, st, a);
}
template <typename FULL>
void launch_units(const BmMoveArgs& a, int unit, bool in_place, dim3 grid, hipStream_t st) {
  if (unit == (int)sizeof(FULL)) launch_pieces<FULL, FULL>(a, in_place, grid, st);
  else if (unit == 2) launch_pieces<FULL, uint16_t>(a, in_place, grid, st);
  else if (unit == 1) launch_pieces<FULL, uint8_t>(a, in_place, grid, st);
  else if constexpr (sizeof(FULL) > 4) launch_pieces<FULL, uint32_t>(a, in_place, grid, st);
}

}  // namespace

extern "C" int cs_beam_reorder(const void* src, void* dst, int64_t outer, int64_t B, int32_t K, int32_t W, int64_t row_bytes,
                               const int64_t src_stride[3], const int64_t dst_stride[3], const int64_t* parents, void* stream) {
  CS_REQUIRE(outer >= 0 && B >= 0 && K >= 1 && W >= 1 && row_bytes >= 0, "bad sizes");
  if (outer == 0 || B == 0 || row_bytes == 0) return CS_OK;
  CS_REQUIRE(src && dst && src_stride && dst_stride && parents, "null argument");
  const bool in_place = src == dst;
  int64_t src_end = row_bytes;
  const int64_t n_src[3] = {outer, B, K}, n_dst[3] = {outer, B, W};
  for (int i = 0; i < 3; ++i) {
    CS_REQUIRE(src_stride[i] >= 0 && dst_stride[i] >= 0, "negative stride");
    src_end += (n_src[i] - 1) * src_stride[i];
  }
  const int64_t dst_end = cs_rows_apart(n_dst, dst_stride, row_bytes);
  CS_REQUIRE(dst_end >= 0, "rows of the destination overlap");
  const char* after = (const char*)(parents + B * W);   // (threads that write rows would do so while others still read their parents)
  CS_REQUIRE(after <= (const char*)dst || (const char*)dst + dst_end <= (const char*)parents, "parents lie in the destination");
  if (in_place) {
    CS_REQUIRE(W == K && K <= 64, "in place: as many chains as before, at most 64");
    for (int i = 0; i < 3; ++i) CS_REQUIRE(n_src[i] == 1 || src_stride[i] == dst_stride[i], "in place: one layout");
  } else {
    CS_REQUIRE((const char*)src + src_end <= (const char*)dst || (const char*)dst + dst_end <= (const char*)src,
               "source and destination overlap");
  }
  BmMoveArgs a;
  a.src = (const char*)src; a.dst = (char*)dst; a.parents = parents;
  a.outer = outer; a.B = B; a.K = K; a.W = W;
  uintptr_t bits = (uintptr_t)src | (uintptr_t)dst | (uintptr_t)row_bytes;
  for (int i = 0; i < 3; ++i) {
    a.ss[i] = src_stride[i]; a.ds[i] = dst_stride[i];
    if (n_src[i] > 1) bits |= (uintptr_t)src_stride[i];
    if (n_dst[i] > 1) bits |= (uintptr_t)dst_stride[i];
  }
  int unit = 1;
  while (unit < 16 && (bits & unit) == 0) unit *= 2;
  const int piece = piece_of(unit, row_bytes, in_place, K);
  unit = unit < piece ? unit : piece;
  a.full = row_bytes / piece;
  a.cols = a.full + (row_bytes - a.full * piece) / unit;
  const int64_t rows = B * (in_place ? 1 : W);
  a.small = rows * a.cols <= UINT32_MAX;
  a.by_cols = cs_div_by(a.small ? a.cols : 1);
  a.by_W = cs_div_by(W);
  const int64_t blocks = (rows * a.cols + 255) / 256;
  CS_REQUIRE(blocks <= INT32_MAX, "too many states for one call");
  // a thread serves several outer indices once that still leaves the chip full
  int64_t split = (8192 + blocks - 1) / blocks;
  split = split < 1 ? 1 : split;
  split = split < outer ? split : outer;
  a.outer_step = split < 65535 ? split : 65535;
  dim3 grid = cs_grid(blocks);
  grid.z = (unsigned)a.outer_step;
  hipStream_t st = (hipStream_t)stream;
  if (piece == 16) launch_units<u32x4>(a, unit, in_place, grid, st);
  else if (piece == 8) launch_units<u32x2>(a, unit, in_place, grid, st);
  else launch_units<uint32_t>(a, unit, in_place, grid, st);
  CS_HIP(hipGetLastError());
  return CS_OK;
}
