// Beam search over chains: the best continuations of all beams of an example, and the states that follow them.  The
// deterministic sibling of the multinomial / systematic resampling (cs_lair.hip, cs_final_resample).
//
// Selection.  s[k,v] = logits[k,v] + (scores[k] - lse[k]), lse the log of the sum of exponentials of the allowed logits
// of beam k: the W largest over (k,v), ties to the lowest k*V + v.  One pass over the logits: a wavefront holds a
// stretch of 2048 of one beam in registers (32 per lane), leaves their maximum, their sum of exponentials relative to it
// and their W best (sorted) in the workspace; a workgroup per example then joins the stretches of every beam, turns the
// kept logits into scores and takes the W best of them.  The normaliser joins before scores of different beams are
// compared, so within a beam a stretch's candidates can be ordered by their logits alone.  Sums and scores are held in
// 64 bits: two beams' candidates are often closer than float32 sums of 10^5 terms are exact, and the indices are to be
// those of the definition.
#include "cs_common.h"

namespace {

constexpr int BM_MAXW = 64;            // candidates per example and per stretch: a lane each
constexpr int BM_LANE = 32;            // logits a lane holds
constexpr int BM_STRETCH = 64 * BM_LANE;
constexpr int BM_LIST = 256;           // preselected logits of a stretch
constexpr int BM_MAXK = 2048;
constexpr int BM_JOIN = 1024;          // threads that join an example, at most
constexpr float BM_LOWEST = -3.402823466e+38f;

struct BmItem { float x; int32_t v; };           // v < 0: none
struct BmStat { double sum; float top; float pad; };

struct BmArgs {
  cs_beam_cfg c;
  const void *scores, *logits;
  const uint8_t *mask, *finished;
  BmStat* stat;     // [B*K*stretches]
  BmItem* item;     // [B*K*stretches][W]
  void* out_scores;
  int64_t *parents, *tokens;
  int32_t stretches;
};

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
  static __device__ __forceinline__ float one(const float* p) { return *p; }
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
  static __device__ __forceinline__ float one(const BmBf16* p) { return __uint_as_float((uint32_t)p->u << 16); }
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
  static __device__ __forceinline__ float one(const _Float16* p) { return (float)*p; }
};

__device__ __forceinline__ float bm_wave_max(float v) {
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ double bm_wave_sum(double v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// 2^(j / 32)
__device__ const double bm_pow32[32] = {
    1, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.6457554781539649,
    1.681792830507429, 1.7186192981224779, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};

// exp(d) for -700 <= d <= 0 as 2^n 2^(j/32) exp(r), 32 n + j the integer nearest to 32 d / ln 2 and |r| <= ln 2 / 64, exp(r) by
// its Taylor polynomial of degree 4 (remainder r^5 / 120 < 1.3e-12): the table-driven method of Tang (1989).  Adding
// 1.5 * 2^52 leaves the integer in the low word.  The table lies in LDS: 32 entries of 8 bytes fill the 64 banks once, so
// no two of them meet in a bank.
__device__ __forceinline__ double bm_exp(double d, const double* pow32) {
  constexpr double MAGIC = 6755399441055744.0;
  const double z = __builtin_fma(d, 46.16624130844683, MAGIC);   // 32 / ln 2
  const int nj = (int)(uint32_t)(uint64_t)__double_as_longlong(z);
  const double r = __builtin_fma(z - MAGIC, -0.02166084939249829, d);   // ln 2 / 32
  const double t = pow32[nj & 31];
  const double tn = __hiloint2double(__double2hiint(t) + ((nj & ~31) << 15), __double2loint(t));
  const double p = __builtin_fma(__builtin_fma(__builtin_fma(__builtin_fma(r, 1.0 / 24, 1.0 / 6), r, 0.5), r, 1.0), r, 1.0);
  return tn * p;
}

// The largest key that at least W lanes reach with theirs (0 if fewer than W lanes have one): bits from the top.
template <typename U>
__device__ __forceinline__ U bm_wave_threshold(U key, int W) {
  U t = 0;
  for (int bit = (int)sizeof(U) * 8 - 1; bit >= 0; --bit) {
    const U u = t | ((U)1 << bit);
    if (__popcll(__ballot(key >= u)) >= W) t = u;
  }
  return t;
}

// One wavefront per stretch.
template <typename T, bool MASK>
__global__ void __launch_bounds__(256) cs_beam_scan_kernel(const BmArgs a) {
  constexpr int N = BmElem<T>::N;      // logits in 16 bytes
  __shared__ BmItem s_list[4][BM_LIST];
  __shared__ double s_pow[32];
  if (threadIdx.x < 32) s_pow[threadIdx.x] = bm_pow32[threadIdx.x];
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t item = (int64_t)blockIdx.x * 4 + wave;
  const int64_t rows = (int64_t)a.c.B * a.c.K;
  const bool live = item < rows * a.stretches;
  const int64_t row = live ? item / a.stretches : 0;
  const int32_t base = live ? (int32_t)(item - row * a.stretches) * BM_STRETCH : 0;
  const int64_t b = row / a.c.K, k = row - b * a.c.K;
  const int W = a.c.W;
  const bool finished = live && a.finished && a.finished[row];
  const int32_t V = (int32_t)a.c.V;
  int n = 0;                           // entries of the list (the same in every lane)
  float top = -__builtin_inff();
  double sum = 0.0;
  if (finished) {                      // its one candidate keeps the beam's score; its logits are not read
    if (lane == 0 && base == 0) s_list[wave][0] = BmItem{0.0f, (int32_t)a.c.end_token};
    n = base == 0 ? 1 : 0;
  } else if (live) {
    const T* p = (const T*)a.logits + b * a.c.logits_stride[0] + k * a.c.logits_stride[1];
    const uint8_t* mk = MASK ? a.mask + b * a.c.mask_stride[0] + k * a.c.mask_stride[1] : nullptr;
    float x[BM_LANE];
#pragma unroll
    for (int j = 0; j < BM_LANE / N; ++j) {
      const int32_t v0 = base + (j * 64 + lane) * N;
      if (v0 + N <= V) {
        uint32_t r[4];
        __builtin_memcpy(r, p + v0, 16);
        BmElem<T>::widen(r, x + j * N);
        if (MASK) {
          uint8_t m[N];
          __builtin_memcpy(m, mk + v0, N);
#pragma unroll
          for (int e = 0; e < N; ++e) x[j * N + e] = m[e] ? x[j * N + e] : -__builtin_inff();
        }
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          x[j * N + e] = v0 + e < V && (!MASK || mk[v0 + e]) ? BmElem<T>::one(p + v0 + e) : -__builtin_inff();
      }
    }
    float best = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < BM_LANE; ++i) best = fmaxf(best, x[i]);   // (a NaN is passed over)
    top = bm_wave_max(best);
    if (a.c.normalise) {
      if (top == __builtin_inff()) {
        sum = __builtin_nan("");
      } else {
        uint64_t nan = 0;
#pragma unroll
        for (int i = 0; i < BM_LANE; ++i) nan |= __ballot(x[i] != x[i]);
        if (top > -__builtin_inff()) {
          const double m = (double)top;
#pragma unroll
          for (int i = 0; i < BM_LANE; ++i) sum += bm_exp(fmax((double)x[i] - m, -690.0), s_pow);   // (less than 1e-299)
          sum = bm_wave_sum(sum);
        }
        if (nan) sum = __builtin_nan("");
      }
    }
    // everything from the W-th largest of the lanes' best on is a candidate
    const uint32_t tk = bm_wave_threshold<uint32_t>(best > -__builtin_inff() ? bm_key(best) : 0u, W);
    float t = tk ? fmaxf(bm_value(tk), BM_LOWEST) : BM_LOWEST;
    const int32_t v_lane = base + lane * N;
#pragma unroll
    for (int i = 0; i < BM_LANE; ++i) {
      const uint64_t m = __ballot(x[i] >= t);
      if (m) {
        const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
        if (x[i] >= t && at < BM_LIST) s_list[wave][at] = BmItem{x[i] + 0.0f, v_lane + (i / N) * 64 * N + i % N};
        n += __popcll(m);
      }
    }
    if (n > BM_LIST) {   // many equal or ascending values: the W-th largest of all, bit by bit
      uint32_t u = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const float f = bm_value(u | (1u << bit));   // (patterns of NaN reach nothing)
        int c = 0;
#pragma unroll
        for (int i = 0; i < BM_LANE; ++i) c += __popcll(__ballot(x[i] >= f));
        if (c >= W) u |= 1u << bit;
      }
      t = bm_value(u);
      n = 0;
#pragma unroll
      for (int i = 0; i < BM_LANE; ++i) {
        const uint64_t m = __ballot(x[i] > t);
        if (x[i] > t) s_list[wave][n + __popcll(m & ((1ull << lane) - 1))] = BmItem{x[i] + 0.0f, v_lane + (i / N) * 64 * N + i % N};
        n += __popcll(m);
      }
      // of those equal to the W-th the first ones
#pragma unroll
      for (int j = 0; j < BM_LANE / N; ++j) {
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
            if (at < W) s_list[wave][at] = BmItem{t + 0.0f, v_lane + j * 64 * N + e};
            ++at;
          }
        n += __shfl(incl, 63);
      }
      n = n < W ? n : W;
    }
  }
  __syncthreads();
  if (!live) return;
  if (lane == 0) a.stat[item] = BmStat{sum, top, 0.0f};
  BmItem* out = a.item + item * W;
  for (int i = lane; i < n; i += 64) {
    const BmItem mine = s_list[wave][i];
    int rank = 0;
    for (int j = 0; j < n; ++j) {
      const BmItem o = s_list[wave][j];
      rank += o.x > mine.x || (o.x == mine.x && o.v < mine.v);
    }
    if (rank < W) out[rank] = mine;
  }
  for (int i = n + lane; i < W; i += 64) out[i] = BmItem{0.0f, -1};
}

// One workgroup per example.
__global__ void __launch_bounds__(BM_JOIN) cs_beam_join_kernel(const BmArgs a, int cap) {
  extern __shared__ char lds[];
  double* s_beam = (double*)lds;                                    // [K] what a kept logit of the beam gets added
  uint64_t* s_key = (uint64_t*)(lds + ((a.c.K * 8 + 15) & ~15));    // [cap]
  int64_t* s_at = (int64_t*)(s_key + cap);                          // [cap] k*V + v
  __shared__ uint64_t s_wave[BM_JOIN / 64];
  __shared__ int64_t s_wave_at[BM_JOIN / 64];
  __shared__ int s_n;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, threads = blockDim.x, waves = threads >> 6;
  const int64_t b = blockIdx.x;
  const int K = a.c.K, W = a.c.W, C = a.stretches;
  const int64_t V = a.c.V;
  const int64_t total = (int64_t)K * C;
  const BmItem* item = a.item + b * total * W;
  // (asked for before the normalisers are formed)
  const BmItem first = tid < total ? item[(int64_t)tid * W] : BmItem{0.0f, -1};
  if (tid == 0) s_n = 0;
  for (int k = wave; k < K; k += waves) {
    const int64_t row = b * K + k;
    double before = 0.0;
    if (a.scores) before = a.c.scores_type == CS_TYPE_F64 ? ((const double*)a.scores)[row] : (double)((const float*)a.scores)[row];
    if (a.c.normalise && !(a.finished && a.finished[row])) {
      const BmStat* st = a.stat + row * C;
      float m = -__builtin_inff();
      for (int c = lane; c < C; c += 64) m = fmaxf(m, st[c].top);
      m = bm_wave_max(m);
      double sum = 0.0;
      if (m > -__builtin_inff())
        for (int c = lane; c < C; c += 64) {
          const BmStat s = st[c];
          // a stretch that holds NaN says so also where nothing else of it counts
          sum += s.top > -__builtin_inff() || s.sum != s.sum ? s.sum * exp((double)fmaxf(s.top, BM_LOWEST) - (double)m) : 0.0;
        }
      sum = bm_wave_sum(sum);
      before -= (double)m + log(sum);     // (+inf, NaN or nothing allowed: NaN, so that no candidate counts)
    }
    if (lane == 0) s_beam[k] = before;
  }
  __syncthreads();
  // the W-th largest among the stretches' best bounds the result from below
  uint64_t best = 0;
  for (int64_t g = tid; g < total; g += threads) {
    const BmItem i = g == tid ? first : item[g * W];
    if (i.v >= 0) {
      const uint64_t key = bm_key64((double)i.x + s_beam[g / C]);
      best = key > best ? key : best;
    }
  }
  const uint64_t t_wave = bm_wave_threshold<uint64_t>(best, W);
  if (lane == 0) s_wave[wave] = t_wave;
  __syncthreads();
  uint64_t t = 1;
  for (int w = 0; w < waves; ++w) t = s_wave[w] > t ? s_wave[w] : t;
  for (int64_t g = tid; g < total; g += threads) {
    const int k = (int)(g / C);
    for (int r = 0; r < W; ++r) {          // sorted: the first that falls short ends the stretch
      const BmItem i = item[g * W + r];
      if (i.v < 0) break;
      const uint64_t key = bm_key64((double)i.x + s_beam[k]);
      if (key < t) break;
      const int at = atomicAdd(&s_n, 1);   // (places in any order: the ranks below depend on the entries alone)
      if (at < cap) { s_key[at] = key; s_at[at] = k * V + i.v; }
    }
  }
  __syncthreads();
  auto put = [&](int w, uint64_t key, int64_t at) {
    const int64_t o = b * W + w;
    const double s = key ? bm_value64(key) : -__builtin_inf();
    if (a.c.scores_type == CS_TYPE_F64) ((double*)a.out_scores)[o] = s;
    else ((float*)a.out_scores)[o] = (float)s;
    a.parents[o] = key ? at / V : (w < K ? w : K - 1);
    a.tokens[o] = key ? at % V : -1;
  };
  const int n = s_n;
  if (n <= cap) {
    for (int i = tid; i < n; i += threads) {
      const uint64_t key = s_key[i];
      const int64_t at = s_at[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += s_key[j] > key || (s_key[j] == key && s_at[j] < at);
      if (rank < W) put(rank, key, at);
    }
    for (int w = n + tid; w < W; w += threads) put(w, 0, 0);
    return;
  }
  // many equal scores: the results one by one, each the best of what comes after the one before
  uint64_t last = ~0ull;
  int64_t last_at = -1;
  for (int w = 0; w < W; ++w) {
    uint64_t key = 0;
    int64_t at = 0;
    for (int64_t g = tid; g < total; g += threads) {
      const int k = (int)(g / C);
      for (int r = 0; r < W; ++r) {
        const BmItem i = item[g * W + r];
        if (i.v < 0) break;
        const uint64_t u = bm_key64((double)i.x + s_beam[k]);
        const int64_t f = k * V + i.v;
        if ((u < last || (u == last && f > last_at)) && (u > key || (u == key && key && f < at))) { key = u; at = f; }
      }
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
    last = key ? key : 0;
    last_at = key ? at : INT64_MAX;
  }
}

template <typename T>
void launch_scan(const BmArgs& a, dim3 grid, hipStream_t st) {
  if (a.mask) hipLaunchKernelGGL((cs_beam_scan_kernel<T, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((cs_beam_scan_kernel<T, false>), grid, dim3(256), 0, st, a);
}

int check_beam(const cs_beam_cfg* c) {
  CS_REQUIRE(c, "null argument");
  CS_REQUIRE(c->B >= 0 && c->K >= 1 && c->K <= BM_MAXK, "1 .. 2048 beams");
  CS_REQUIRE(c->V >= 1 && c->V <= (int64_t)INT32_MAX - 2 * BM_STRETCH, "bad number of values");
  CS_REQUIRE(c->W >= 1 && c->W <= BM_MAXW, "width must be 1 .. 64");
  CS_REQUIRE(c->logits_type == CS_TYPE_F32 || c->logits_type == CS_TYPE_BF16 || c->logits_type == CS_TYPE_F16,
             "logits are float32, bfloat16 or float16");
  CS_REQUIRE(c->scores_type == CS_TYPE_F32 || c->scores_type == CS_TYPE_F64, "scores are float32 or float64");
  const int64_t stretches = (c->V + BM_STRETCH - 1) / BM_STRETCH;
  CS_REQUIRE((int64_t)c->B * c->K <= ((int64_t)INT32_MAX * 4) / stretches, "too many logits for one call");
  return CS_OK;
}

}  // namespace

extern "C" int64_t cs_beam_select_workspace(const cs_beam_cfg* c) {
  if (check_beam(c)) return -1;
  const int64_t stretches = (c->V + BM_STRETCH - 1) / BM_STRETCH;
  return (int64_t)c->B * c->K * stretches * (int64_t)(sizeof(BmStat) + c->W * sizeof(BmItem));
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
  a.stretches = (int32_t)((c->V + BM_STRETCH - 1) / BM_STRETCH);
  const int64_t items = (int64_t)c->B * c->K * a.stretches;
  a.stat = (BmStat*)workspace;
  a.item = (BmItem*)(a.stat + items);
  a.out_scores = out_scores; a.parents = parents; a.tokens = tokens;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)((items + 3) / 4));
  if (c->logits_type == CS_TYPE_F32) launch_scan<float>(a, grid, st);
  else if (c->logits_type == CS_TYPE_BF16) launch_scan<BmBf16>(a, grid, st);
  else launch_scan<_Float16>(a, grid, st);
  CS_HIP(hipGetLastError());
  // a place for W candidates of each of W stretches, up to 32 KB
  int cap = c->W * c->W;
  cap = cap < 256 ? 256 : cap > 2048 ? 2048 : cap;
  // a thread per stretch, as far as that goes
  const int64_t total = (int64_t)c->K * a.stretches;
  const int threads = total <= 64 && c->K <= 4 ? 64 : total <= 256 ? 256 : BM_JOIN;
  hipLaunchKernelGGL(cs_beam_join_kernel, dim3((unsigned)c->B), dim3(threads), (size_t)(((c->K * 8 + 15) & ~15) + cap * 16), st, a,
                     cap);
  CS_HIP(hipGetLastError());
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
  int64_t outer, B, cols;              // cols: vectors of a row
  int64_t ss[3], ds[3];                // bytes between outer / example / chain
  int32_t K, W;
  int64_t outer_step;                  // a thread serves every outer_step-th outer index
};

// out of place: a thread per vector of a destination row, over its outer indices
template <typename VEC>
__global__ void __launch_bounds__(256) cs_beam_gather_kernel(const BmMoveArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.B * a.W * a.cols) return;
  const int64_t bw = i / a.cols, col = i - bw * a.cols;
  const int64_t p = a.parents[bw];
  if (p < 0 || p >= a.K) return;
  const int64_t b = bw / a.W, w = bw - b * a.W;
  const char* s = a.src + b * a.ss[1] + p * a.ss[2] + col * sizeof(VEC);
  char* d = a.dst + b * a.ds[1] + w * a.ds[2] + col * sizeof(VEC);
  for (int64_t o = blockIdx.y; o < a.outer; o += a.outer_step)
    *(VEC*)(d + o * a.ds[0]) = *(const VEC*)(s + o * a.ss[0]);
}

// in place: a thread owns one vector column of all K rows of an example, so it reads every row it needs before it
// writes any; rows that keep their place are neither read nor written
template <typename VEC, int KMAX>
__global__ void __launch_bounds__(256) cs_beam_inplace_kernel(const BmMoveArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.B * a.cols) return;
  const int64_t b = i / a.cols, col = i - b * a.cols;
  int parent[KMAX];
#pragma unroll
  for (int k = 0; k < KMAX; ++k) {
    const int64_t p = k < a.K ? a.parents[b * a.K + k] : -1;
    parent[k] = p < 0 || p >= a.K || p == k ? -1 : (int)p;
  }
  char* d = a.dst + b * a.ds[1] + col * sizeof(VEC);
  for (int64_t o = blockIdx.y; o < a.outer; o += a.outer_step) {
    VEC v[KMAX];
#pragma unroll
    for (int k = 0; k < KMAX; ++k)
      if (parent[k] >= 0) v[k] = *(const VEC*)(d + o * a.ds[0] + parent[k] * a.ds[2]);
#pragma unroll
    for (int k = 0; k < KMAX; ++k)
      if (parent[k] >= 0) *(VEC*)(d + o * a.ds[0] + k * a.ds[2]) = v[k];
  }
}

template <typename VEC>
void launch_move(const BmMoveArgs& a, bool in_place, dim3 grid, hipStream_t st) {
  if (!in_place) hipLaunchKernelGGL(cs_beam_gather_kernel<VEC>, grid, dim3(256), 0, st, a);
  else if (a.K <= 4) hipLaunchKernelGGL((cs_beam_inplace_kernel<VEC, 4>), grid, dim3(256), 0, st, a);
  else if (a.K <= 8) hipLaunchKernelGGL((cs_beam_inplace_kernel<VEC, 8>), grid, dim3(256), 0, st, a);
  else if (a.K <= 16) hipLaunchKernelGGL((cs_beam_inplace_kernel<VEC, 16>), grid, dim3(256), 0, st, a);
  else if (a.K <= 32) hipLaunchKernelGGL((cs_beam_inplace_kernel<VEC, 32>), grid, dim3(256), 0, st, a);
  else if constexpr (sizeof(VEC) <= 8) hipLaunchKernelGGL((cs_beam_inplace_kernel<VEC, 64>), grid, dim3(256), 0, st, a);
}

}  // namespace

extern "C" int cs_beam_reorder(const void* src, void* dst, int64_t outer, int64_t B, int32_t K, int32_t W, int64_t row_bytes,
                               const int64_t src_stride[3], const int64_t dst_stride[3], const int64_t* parents, void* stream) {
  CS_REQUIRE(outer >= 0 && B >= 0 && K >= 1 && W >= 1 && row_bytes >= 0, "bad sizes");
  if (outer == 0 || B == 0 || row_bytes == 0) return CS_OK;
  CS_REQUIRE(src && dst && src_stride && dst_stride && parents, "null argument");
  const bool in_place = src == dst;
  int64_t src_end = row_bytes, dst_end = row_bytes;
  const int64_t n_src[3] = {outer, B, K}, n_dst[3] = {outer, B, W};
  for (int i = 0; i < 3; ++i) {
    CS_REQUIRE(src_stride[i] >= 0 && dst_stride[i] >= 0, "negative stride");
    src_end += (n_src[i] - 1) * src_stride[i];
  }
  // the destination's rows must not meet: from the closest axis on, every stride clears what lies within
  int order[3] = {0, 1, 2};
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j)
      if (dst_stride[order[j]] > dst_stride[order[j + 1]]) { const int t = order[j]; order[j] = order[j + 1]; order[j + 1] = t; }
  for (int i = 0; i < 3; ++i)
    if (n_dst[order[i]] > 1) {
      CS_REQUIRE(dst_stride[order[i]] >= dst_end, "rows of the destination overlap");
      dst_end += (n_dst[order[i]] - 1) * dst_stride[order[i]];
    }
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
  // (64 rows of 16-byte columns would not fit a thread's registers)
  const int vec = (bits & 15) == 0 && !(in_place && K > 32) ? 16 : (bits & 7) == 0 ? 8 : (bits & 3) == 0 ? 4 : (bits & 1) == 0 ? 2 : 1;
  a.cols = row_bytes / vec;
  const int64_t blocks = (B * (in_place ? 1 : W) * a.cols + 255) / 256;
  CS_REQUIRE(blocks <= INT32_MAX, "too many states for one call");
  // a thread serves several outer indices once that still leaves the chip full
  int64_t split = (8192 + blocks - 1) / blocks;
  split = split < 1 ? 1 : split;
  split = split < outer ? split : outer;
  a.outer_step = split < 65535 ? split : 65535;
  const dim3 grid((unsigned)blocks, (unsigned)a.outer_step);
  hipStream_t st = (hipStream_t)stream;
  if (vec == 16) launch_move<u32x4>(a, in_place, grid, st);
  else if (vec == 8) launch_move<u32x2>(a, in_place, grid, st);
  else if (vec == 4) launch_move<uint32_t>(a, in_place, grid, st);
  else if (vec == 2) launch_move<uint16_t>(a, in_place, grid, st);
  else launch_move<uint8_t>(a, in_place, grid, st);
  CS_HIP(hipGetLastError());
  return CS_OK;
}
