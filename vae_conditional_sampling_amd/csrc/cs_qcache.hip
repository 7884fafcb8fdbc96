// History ring in 8 or 4 bits: past states [T,B,K,D] quantised as they are written and read back by slot and chain.  The
// counterpart of the float32 and uint8 rings (cs_history_enqueue, cs_history_concat) for real-valued data.
//
// A state is one record: its codes, then the scales of its groups (consecutive values along D), padded to 16 bytes.
// Codes and scales lie together because states are fetched singly, by a slot per chain: a MiniBooNE state (D = 43) in 8
// bits is one record of 48 bytes instead of a row of 172 and is fetched with one or two cache lines.
//   int8   scale s = max(fl32(largest finite magnitude / 127), 2^-126), code = the integer nearest to the real quotient
//          x / s, ties to even; -128 marks a value that was not finite (it reads as NaN).
//   mxfp8  e4m3 elements, mxfp4 e2m1 elements of OCP Microscaling: scale 2^e as an e + 127 byte, groups of 32.  e is the
//          smallest with the largest finite magnitude within the elements' range, so that no value is clipped and every
//          rounding is off by at most half a step.  Not finite: the NaN of e4m3; e2m1 has none, there the group's
//          scale becomes 255 and the group reads as NaN.
// A lane holds 8 values, G / 8 neighbouring lanes share a group's maximum; both directions are bound by memory.
#include "cs_common.h"
#include "cs_div.h"

namespace {

constexpr int QC_LANE = 8;     // values a lane holds

struct QcArgs {
  cs_qcache c;
  int64_t record;              // bytes
  int32_t code_bytes;          // of a record, rounded up to 4
  int32_t lanes;               // lanes of a row: write: groups * G / 8; read: D / 8, rounded up
  int32_t rows_per_block;
  int32_t lg_shift;            // 2^lg_shift lanes share a group's scale
  uint32_t rows;               // rows of the call, below 2^31
  CsDiv by_lanes, by_chains, by_inner, by_T;   // lanes; B * K (write) or B * J (read); K or J; T
  const void* x;               // write
  void* out;                   // read
  int64_t stride[3];
  int64_t start0;
  const int64_t *start, *count, *slots, *from;
};

struct QcBf16 { uint16_t u; };
__device__ __forceinline__ float qc_float(float v) { return v; }
__device__ __forceinline__ float qc_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float qc_float(QcBf16 v) { return __uint_as_float((uint32_t)v.u << 16); }
// The largest finite value of the type that is read: what rounds up beyond it (a code to the next power of two, the scale of the
// very largest states) is cut to it, so that a finite state reads as a finite value.
template <typename T> struct QcMost { static constexpr float value = 3.402823466e+38f; static constexpr int e = 127; };   // (2 - ulp) 2^e
template <> struct QcMost<_Float16> { static constexpr float value = 65504.0f; static constexpr int e = 15; };
template <> struct QcMost<QcBf16> { static constexpr float value = 3.389531389e+38f; static constexpr int e = 127; };
__device__ __forceinline__ void qc_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void qc_store(_Float16* p, float v) { *p = (_Float16)v; }
__device__ __forceinline__ void qc_store(QcBf16* p, float v) {   // nearest, ties to even
  const uint32_t u = __float_as_uint(v);
  p->u = (uint16_t)(v != v ? 0x7fc0u : (u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}

// The largest of the lanes of a group (lg = 1 to 16 neighbouring lanes): exchanges within quads, then the mirrored other
// half of 8 and of 16 lanes, whose halves are of one value by then.
__device__ __forceinline__ uint32_t qc_group_max(uint32_t v, int lg) {
#define CS_STEP(CTRL_)                                                                                        \
  {                                                                                                           \
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL_, 0xf, 0xf, false);         \
    v = o > v ? o : v;                                                                                        \
  }
  if (lg > 1) CS_STEP(0xb1)              // quad_perm: 1 0 3 2
  if (lg > 2) CS_STEP(0x4e)              // quad_perm: 2 3 0 1
  if (lg > 4) CS_STEP(0x141)             // row_half_mirror
  if (lg > 8) CS_STEP(0x140)             // row_mirror
#undef CS_STEP
  return v;
}

// Codes of 8 values of a group whose largest finite magnitude is `top`; `fine`: all of the GROUP's values are finite (PLAIN:
// those of every group of the wavefront).  The scale goes to `scale` (int8: a float's bits, else the byte).
template <int FMT, bool PLAIN>
__device__ __forceinline__ void qc_encode(const float* x, float top, bool fine, uint32_t* codes, uint32_t* scale) {
  auto finite = [](float v) { return PLAIN || __builtin_fabsf(v) <= 3.402823466e+38f; };
  if (FMT == CS_QFMT_INT8) {
    // top / 127 as division rounds it: one remainder corrects the product with fl(1/127) (Markstein 1990; below 127 * 2^-126, where
    // remainders would not be exact, the scale does not depend on it)
    constexpr float INV127 = 1.0f / 127.0f;
    const float q127 = top * INV127;
    const float s = fmaxf(__builtin_fmaf(__builtin_fmaf(-q127, 127.0f, top), INV127, q127), 1.17549435e-38f);
    const float inv = __builtin_amdgcn_rcpf(s);   // (a unit in the last place off at most)
    float q[QC_LANE];
    bool near = false;
#pragma unroll
    for (int i = 0; i < QC_LANE; ++i) {
      const float v = (finite(x[i]) ? x[i] : 0.0f) * inv;
      q[i] = __builtin_rintf(v);
      near = near || __builtin_fabsf(v - q[i]) > 0.4999f;
    }
    if (__ballot(near)) {
      // v is off by less than 3e-5, so these alone can be beside the nearest integer of the real quotient: the remainder
      // x - q s is exact (a multiple of the last place of s or x, below 2^24 of them) and says so
#pragma unroll
      for (int i = 0; i < QC_LANE; ++i) {
        const float v = finite(x[i]) ? x[i] : 0.0f;
        const float r = 2.0f * __builtin_fmaf(-q[i], s, v);
        const float away = __builtin_fabsf(r);
        const bool odd = ((int)q[i] & 1) != 0;
        if (away > s || (away == s && odd)) q[i] += r > 0.0f ? 1.0f : -1.0f;
        q[i] = fminf(fmaxf(q[i], -127.0f), 127.0f);
      }
    }
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < QC_LANE; ++i) {
      const uint32_t c = finite(x[i]) ? (uint32_t)(int)q[i] & 0xffu : 0x80u;
      w[i >> 2] |= c << (8 * (i & 3));
    }
    codes[0] = w[0]; codes[1] = w[1];
    *scale = __float_as_uint(s);
    return;
  }
  const float largest = FMT == CS_QFMT_MXFP8 ? 0.875f : 0.75f;       // 448 = 0.875 * 2^9, 6 = 0.75 * 2^3
  int e = -127;
  if (top > 0.0f) {
    e = __builtin_amdgcn_frexp_expf(top) - (FMT == CS_QFMT_MXFP8 ? 9 : 3) + (__builtin_amdgcn_frexp_mantf(top) > largest ? 1 : 0);
    e = e < -127 ? -127 : e;
  }
  float y[QC_LANE];
#pragma unroll
  for (int i = 0; i < QC_LANE; ++i)
    y[i] = finite(x[i]) ? __builtin_amdgcn_ldexpf(x[i], -e) : (FMT == CS_QFMT_MXFP8 ? __builtin_nanf("") : 0.0f);
  if (FMT == CS_QFMT_MXFP8) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], w, true);
      codes[h] = (uint32_t)w;
    }
  } else {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.0f, 3);
    codes[0] = w;
  }
  *scale = FMT == CS_QFMT_MXFP4 && !fine ? 255u : (uint32_t)(e + 127);
}

template <int FMT, typename T>
__device__ __forceinline__ void qc_decode(const uint32_t* codes, uint32_t scale, float* v) {
  constexpr float most = QcMost<T>::value;
  typedef float f2 __attribute__((ext_vector_type(2)));
  if (FMT == CS_QFMT_INT8) {
    const float s = __uint_as_float(scale);
#pragma unroll
    for (int i = 0; i < QC_LANE; ++i) {
      const int q = (int8_t)(codes[i >> 2] >> (8 * (i & 3)));
      const float p = fminf(fmaxf((float)q * s, -most), most);
      v[i] = q == -128 ? __builtin_nanf("") : p;
    }
    return;
  }
  const int e = (int)scale - 127;
  if (FMT == CS_QFMT_MXFP8) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[h], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[h], true);
      v[4 * h] = a.x; v[4 * h + 1] = a.y; v[4 * h + 2] = b.x; v[4 * h + 3] = b.y;
    }
  } else {
    const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], 1.0f, 1),
             c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], 1.0f, 3);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
  }
#pragma unroll
  for (int i = 0; i < QC_LANE; ++i) v[i] = __builtin_amdgcn_ldexpf(v[i], e);
  // elements end at 1.75 * 2^8 and 1.5 * 2^2: no scale up to this one leaves the range
  if (__builtin_expect(e > QcMost<T>::e - (FMT == CS_QFMT_MXFP8 ? 8 : 2), 0)) {
#pragma unroll
    for (int i = 0; i < QC_LANE; ++i)   // (a NaN stays: fmax and fmin would pass it over)
      v[i] = scale == 255u ? __builtin_nanf("") : __builtin_fabsf(v[i]) > most ? __builtin_copysignf(most, v[i]) : v[i];
  }
}

// the slot of step i of a chain of a call that runs from `start` on; -1: not in the call
__device__ __forceinline__ int32_t qc_slot(const QcArgs& a, uint32_t i, uint32_t chain) {
  const uint32_t T = a.by_T.d;
  // (both asked for at once)
  const int64_t count = a.count ? a.count[chain] : INT64_MAX;
  const int64_t far = a.start ? a.start[chain] : a.start0;      // (start0 is below T)
  if ((int64_t)i >= count || far < 0) return -1;
  uint32_t s = far < (int64_t)T ? (uint32_t)far : (uint32_t)(far % (int64_t)T);
  s += i - cs_div(i, a.by_T) * T;
  return (int32_t)(s >= T ? s - T : s);
}

// 8 values from / to addresses aligned to the type alone (the hardware takes any address)
template <typename T>
__device__ __forceinline__ void qc_load8(const T* p, float* v) {
  T r[QC_LANE];
  __builtin_memcpy(r, p, sizeof(r));
#pragma unroll
  for (int e = 0; e < QC_LANE; ++e) v[e] = qc_float(r[e]);
}
template <typename T>
__device__ __forceinline__ void qc_store8(T* p, const float* v) {
  T r[QC_LANE];
#pragma unroll
  for (int e = 0; e < QC_LANE; ++e) qc_store(r + e, v[e]);
  __builtin_memcpy(p, r, sizeof(r));
}

// Bound by memory: 134 M bfloat16 values to mxfp8 (406 MB) take 86 us, 4.7 TB/s, the rate of a copy.
template <int FMT, typename T>
__global__ void __launch_bounds__(256) cs_qcache_write_kernel(const QcArgs a) {
  const int ry = (int)cs_div(threadIdx.x, a.by_lanes);
  const uint32_t row = cs_block() * (uint32_t)a.rows_per_block + (uint32_t)ry;
  if (ry >= a.rows_per_block || row >= a.rows) return;
  const uint32_t i = cs_div(row, a.by_chains), chain = row - i * a.by_chains.d;
  const int32_t slot = qc_slot(a, i, chain);
  if (slot < 0) return;                  // (all lanes of a row stay or leave, so the lanes of a group stay together)
  const uint32_t b = cs_div(chain, a.by_inner), k = chain - b * a.by_inner.d;
  const T* x = (const T*)a.x + i * a.stride[0] + b * a.stride[1] + k * a.stride[2];
  char* rec = (char*)a.c.data + ((int64_t)slot * a.by_chains.d + chain) * a.record;
  const int D = a.c.D, lg = 1 << a.lg_shift;
  // (lanes of a row: a multiple of the lanes of a group, which divide 64)
  for (int l = threadIdx.x - ry * a.lanes; l < a.lanes; l += 256) {
    const int d0 = l * QC_LANE;
    float v[QC_LANE];
    if (d0 + QC_LANE <= D) {
      qc_load8(x + d0, v);
    } else {
#pragma unroll
      for (int e = 0; e < QC_LANE; ++e) v[e] = d0 + e < D ? qc_float(x[d0 + e]) : 0.0f;
    }
    // (magnitudes order as their bits do; infinities and NaN lie above all others)
    constexpr uint32_t INFBITS = 0x7f800000u;
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < QC_LANE; ++e) {
      const uint32_t m = __float_as_uint(v[e]) & 0x7fffffffu;
      top = m > top ? m : top;
    }
    top = qc_group_max(top, lg);
    uint32_t codes[2] = {0, 0}, scale = 0;
    if (__ballot(top >= INFBITS) == 0) {
      qc_encode<FMT, true>(v, __uint_as_float(top), true, codes, &scale);
    } else {
      const bool fine = top < INFBITS;
      top = 0;
#pragma unroll
      for (int e = 0; e < QC_LANE; ++e) {
        const uint32_t m = __float_as_uint(v[e]) & 0x7fffffffu;
        top = m > top && m < INFBITS ? m : top;
      }
      top = qc_group_max(top, lg);
      qc_encode<FMT, false>(v, __uint_as_float(top), fine, codes, &scale);
    }
    const int c0 = FMT == CS_QFMT_MXFP4 ? d0 / 2 : d0;
    if (c0 < a.code_bytes) *(uint32_t*)(rec + c0) = codes[0];
    if (FMT != CS_QFMT_MXFP4 && c0 + 4 < a.code_bytes) *(uint32_t*)(rec + c0 + 4) = codes[1];
    if ((l & (lg - 1)) == 0) {
      if (FMT == CS_QFMT_INT8) *(uint32_t*)(rec + a.code_bytes + 4 * (l >> a.lg_shift)) = scale;
      else *(uint8_t*)(rec + a.code_bytes + (l >> a.lg_shift)) = (uint8_t)scale;
    }
  }
}

// R rows per lane, rows_per_block apart: their index loads, then their records, are under way together, where a call has
// rows enough to fill the chip even so (a lane's chain of slot, record and store is some 5 us long): 134 M values from mxfp8 to
// bfloat16 (406 MB) in 92 us with R = 4, 108 with 1.
// PACKED: the rows of the call follow each other in `out` and their length is no multiple of 8 values.  Then the lanes' pieces
// of a row would be stored in up to 8 parts each, every one of them touching all lines of the block's rows; the block's
// rows are put together in LDS instead and stored as one run of 16-byte pieces: 524288 rows of 21 float32 from scattered records
// in 18.5 us, 30 without.  Rows of more than 16 lanes gain nothing by it.
template <int FMT, typename T, int R, bool PACKED>
__global__ void __launch_bounds__(256) cs_qcache_read_kernel(const QcArgs a) {
  extern __shared__ __align__(16) char lds[];
  T* s_out = (T*)lds;                  // [R * rows_per_block][D]
  const int ry = (int)cs_div(threadIdx.x, a.by_lanes);
  const uint32_t row0 = cs_block() * (uint32_t)(R * a.rows_per_block);
  if (row0 >= a.rows) return;
  const char* rec[R];
  T* out[R];
  bool live[R], there[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t row = row0 + r * a.rows_per_block + ry;
    live[r] = ry < a.rows_per_block && row < a.rows;
    const uint32_t at = live[r] ? row : 0, i = cs_div(at, a.by_chains), chain = at - i * a.by_chains.d;
    const uint32_t b = cs_div(chain, a.by_inner), j = chain - b * a.by_inner.d;
    const int64_t slot = a.slots ? a.slots[at] : qc_slot(a, i, chain);
    const int64_t k = a.from ? a.from[at] : j;
    there[r] = slot >= 0 && slot < a.c.T && k >= 0 && k < a.c.K;
    rec[r] = (const char*)a.c.data + (there[r] ? ((slot * a.c.B + b) * a.c.K + k) * a.record : 0);
    out[r] = PACKED ? s_out + (r * a.rows_per_block + ry) * a.c.D
                    : (T*)a.out + i * a.stride[0] + b * a.stride[1] + j * a.stride[2];
  }
  const int D = a.c.D;
  for (int l = threadIdx.x - ry * a.lanes; l < a.lanes; l += 256) {
    const int d0 = l * QC_LANE;
    if (d0 >= D) break;
    uint32_t codes[R][2], scale[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {   // (the first record's bytes stand in for those of a row that does not exist)
      const int c0 = FMT == CS_QFMT_MXFP4 ? d0 / 2 : d0;
      codes[r][0] = *(const uint32_t*)(rec[r] + c0);
      codes[r][1] = FMT != CS_QFMT_MXFP4 && c0 + 4 < a.code_bytes ? *(const uint32_t*)(rec[r] + c0 + 4) : 0;
      scale[r] = FMT == CS_QFMT_INT8 ? *(const uint32_t*)(rec[r] + a.code_bytes + 4 * (l >> a.lg_shift))
                                    : *(const uint8_t*)(rec[r] + a.code_bytes + (l >> a.lg_shift));
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float v[QC_LANE];
      qc_decode<FMT, T>(codes[r], scale[r], v);
#pragma unroll
      for (int e = 0; e < QC_LANE; ++e) v[e] = there[r] ? v[e] : 0.0f;
      if (!live[r]) continue;
      if (d0 + QC_LANE <= D) {
        qc_store8(out[r] + d0, v);
      } else {
#pragma unroll
        for (int e = 0; e < QC_LANE; ++e)
          if (d0 + e < D) qc_store(out[r] + d0 + e, v[e]);
      }
    }
  }
  if (PACKED) {
    __syncthreads();
    const uint32_t rows = a.rows - row0 < (uint32_t)(R * a.rows_per_block) ? a.rows - row0 : (uint32_t)(R * a.rows_per_block);
    const int n = (int)rows * D;
    T* to = (T*)a.out + (int64_t)row0 * D;
    constexpr int E = 16 / (int)sizeof(T);
    for (int e = threadIdx.x * E; e < n; e += 256 * E) {
      if (e + E <= n) {
        uint32_t w[4];
        __builtin_memcpy(w, __builtin_assume_aligned(s_out + e, 16), 16);
        __builtin_memcpy(to + e, w, 16);
      } else {
        for (int f = e; f < n; ++f) to[f] = s_out[f];
      }
    }
  }
}

int64_t code_bytes_of(int fmt, int64_t D) {
  const int64_t n = fmt == CS_QFMT_MXFP4 ? (D + 1) / 2 : D;
  return (n + 3) / 4 * 4;
}

int check_qcache(const cs_qcache* c) {
  CS_REQUIRE(c, "null argument");
  CS_REQUIRE(c->T >= 1 && c->T <= INT32_MAX && c->B >= 0 && c->K >= 1 && c->D >= 1, "bad sizes");
  CS_REQUIRE(c->fmt == CS_QFMT_INT8 || c->fmt == CS_QFMT_MXFP8 || c->fmt == CS_QFMT_MXFP4, "unknown format");
  if (c->fmt == CS_QFMT_INT8) CS_REQUIRE(c->group == 32 || c->group == 64 || c->group == 128, "int8: groups of 32, 64 or 128");
  else CS_REQUIRE(c->group == 32, "mxfp8 / mxfp4: groups of 32");
  CS_REQUIRE(c->D <= (1 << 24), "rows too long");
  return CS_OK;
}

template <bool WRITE, int FMT, typename T>
void launch_rows(const QcArgs& a, int R, bool packed, dim3 grid, hipStream_t st) {
  const size_t lds = (size_t)a.rows_per_block * a.c.D * sizeof(T);   // (at most 256 * 8 values)
  if constexpr (WRITE) {
    hipLaunchKernelGGL((cs_qcache_write_kernel<FMT, T>), grid, dim3(256), 0, st, a);
  } else {
    if (packed) hipLaunchKernelGGL((cs_qcache_read_kernel<FMT, T, 1, true>), grid, dim3(256), lds, st, a);
    else if (R == 4) hipLaunchKernelGGL((cs_qcache_read_kernel<FMT, T, 4, false>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((cs_qcache_read_kernel<FMT, T, 1, false>), grid, dim3(256), 0, st, a);
  }
}
template <bool WRITE, int FMT>
void launch_type(const QcArgs& a, int type, int R, bool packed, dim3 grid, hipStream_t st) {
  if (type == CS_TYPE_F32) launch_rows<WRITE, FMT, float>(a, R, packed, grid, st);
  else if (type == CS_TYPE_BF16) launch_rows<WRITE, FMT, QcBf16>(a, R, packed, grid, st);
  else launch_rows<WRITE, FMT, _Float16>(a, R, packed, grid, st);
}

bool apart(const void* p, int64_t p_bytes, const void* q, int64_t q_bytes) {
  return !p || !q || (const char*)p + p_bytes <= (const char*)q || (const char*)q + q_bytes <= (const char*)p;
}

// n steps of B * inner rows
template <bool WRITE>
int launch(QcArgs& a, int64_t n, int32_t inner, int64_t start0, int type, hipStream_t st) {
  const cs_qcache& c = a.c;
  CS_REQUIRE(c.B <= INT32_MAX / inner && n <= INT32_MAX / (c.B * inner), "2^31 states or more in one call");
  a.rows = (uint32_t)(n * c.B * inner);
  a.by_chains = cs_div_by(c.B * inner);
  a.by_inner = cs_div_by(inner);
  a.by_T = cs_div_by(c.T);
  a.start0 = start0 % c.T;
  CS_REQUIRE(type == CS_TYPE_F32 || type == CS_TYPE_BF16 || type == CS_TYPE_F16, "states are float32, bfloat16 or float16");
  CS_REQUIRE(((uintptr_t)c.data & 15) == 0, "the ring must be 16-byte aligned");
  a.record = cs_qcache_record_bytes(c.fmt, c.group, c.D);
  a.code_bytes = (int32_t)code_bytes_of(c.fmt, c.D);
  // what is written is neither written twice nor read by other threads
  const int64_t sizes[3] = {n, c.B, inner}, size = type == CS_TYPE_F32 ? 4 : 2;
  const int64_t ring = c.T * c.B * c.K * a.record, indices = (int64_t)a.rows * 8;
  int64_t end = c.D;
  for (int i = 0; i < 3; ++i) {
    CS_REQUIRE(a.stride[i] >= 0, "negative stride");
    end += (sizes[i] - 1) * a.stride[i];
  }
  if (WRITE) {
    CS_REQUIRE(apart(a.x, end * size, c.data, ring), "states lie in the ring");
  } else {
    CS_REQUIRE(cs_rows_apart(sizes, a.stride, c.D) >= 0, "rows of the output overlap");
    CS_REQUIRE(apart(a.out, end * size, c.data, ring) && apart(a.out, end * size, a.slots, indices) &&
               apart(a.out, end * size, a.from, indices), "the output lies in what is read");
  }
  if (WRITE)
    while (a.c.group > QC_LANE && c.D <= a.c.group / 2) a.c.group /= 2;   // (a row of one group, cut to what it holds)
  a.lanes = WRITE ? (c.D + a.c.group - 1) / a.c.group * (a.c.group / QC_LANE) : (c.D + QC_LANE - 1) / QC_LANE;
  a.lg_shift = __builtin_ctz((unsigned)(a.c.group / QC_LANE));   // (groups are powers of two)
  a.by_lanes = cs_div_by(a.lanes);
  a.rows_per_block = a.lanes >= 256 ? 1 : 256 / a.lanes;
  const uint32_t blocks = (a.rows + a.rows_per_block - 1) / a.rows_per_block;
  const bool packed = !WRITE && c.D % QC_LANE != 0 && a.lanes <= 16 && a.stride[2] == c.D && a.stride[1] == (int64_t)inner * c.D &&
                      (n == 1 || a.stride[0] == c.B * inner * c.D);
  const int R = WRITE || packed || blocks < 8192 ? 1 : 4;
  const dim3 grid = cs_grid((blocks + R - 1) / R);
  if (c.fmt == CS_QFMT_INT8) launch_type<WRITE, CS_QFMT_INT8>(a, type, R, packed, grid, st);
  else if (c.fmt == CS_QFMT_MXFP8) launch_type<WRITE, CS_QFMT_MXFP8>(a, type, R, packed, grid, st);
  else launch_type<WRITE, CS_QFMT_MXFP4>(a, type, R, packed, grid, st);
  CS_HIP(hipGetLastError());
  return CS_OK;
}

}  // namespace

extern "C" int64_t cs_qcache_record_bytes(int32_t fmt, int32_t group, int32_t D) {
  const cs_qcache c = {nullptr, 1, 1, 1, D, fmt, group};
  if (check_qcache(&c)) return -1;
  const int64_t groups = (D + group - 1) / group;
  return (code_bytes_of(fmt, D) + groups * (fmt == CS_QFMT_INT8 ? 4 : 1) + 15) / 16 * 16;
}

extern "C" int cs_qcache_write(const cs_qcache* c, const void* X, int32_t x_type, int64_t n, const int64_t x_stride[3],
                               const int64_t* start, int64_t start0, const int64_t* count, void* stream) {
  if (int rc = check_qcache(c)) return rc;
  CS_REQUIRE(n >= 0 && n <= c->T, "at most T states of a chain per call");
  CS_REQUIRE(start || start0 >= 0, "negative start");
  if (n == 0 || c->B == 0) return CS_OK;
  CS_REQUIRE(c->data && X && x_stride, "null argument");
  QcArgs a = {};
  a.c = *c;
  a.x = X; a.start = start; a.count = count;
  for (int i = 0; i < 3; ++i) a.stride[i] = x_stride[i];
  return launch<true>(a, n, c->K, start ? 0 : start0, x_type, (hipStream_t)stream);
}

extern "C" int cs_qcache_read(const cs_qcache* c, const int64_t* slots, int64_t start0, const int64_t* chains, int64_t N, int32_t J,
                              void* out, int32_t out_type, const int64_t out_stride[3], void* stream) {
  if (int rc = check_qcache(c)) return rc;
  CS_REQUIRE(N >= 0 && J >= 1, "bad sizes");
  CS_REQUIRE(chains || J == c->K, "without chains a row is read of every chain");
  CS_REQUIRE(slots || start0 >= 0, "negative start");
  if (N == 0 || c->B == 0) return CS_OK;
  CS_REQUIRE(c->data && out && out_stride, "null argument");
  QcArgs a = {};
  a.c = *c;
  a.out = out; a.slots = slots; a.from = chains;
  for (int i = 0; i < 3; ++i) a.stride[i] = out_stride[i];
  return launch<false>(a, N, J, slots ? 0 : start0, out_type, (hipStream_t)stream);
}
