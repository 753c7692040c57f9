// Device code shared by the operators on rows of class logits: 16-byte packs,
// rows held in registers, the rules of a row, wave reductions.
#pragma once

#include <cfloat>

#include "device_math.h"
#include "logits.h"

namespace ppocr {

constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------- reductions
// Lanes where v holds (the compare's own result; HIP's __ballot makes an
// integer of it first).
__device__ __forceinline__ uint64_t lanes_where(bool v) { return __builtin_amdgcn_ballot_w64(v); }

// Data-parallel moves within a wave (row shifts by 1, 2, 4 and 8, then the
// last lane of 16 and of 32 to the lanes behind): a few cycles a step, where
// a shuffle goes through LDS.  The whole wave must be active.  Lanes without
// a source keep `old`.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_move(int old, int v) {
  return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xf, false);
}
template <typename F>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t v, uint32_t none, F&& f) {
#define STEP(CTRL, ROWS) v = f(v, (uint32_t)dpp_move<CTRL, ROWS>((int)none, (int)v))
  STEP(0x111, 0xf);
  STEP(0x112, 0xf);
  STEP(0x114, 0xf);
  STEP(0x118, 0xf);
  STEP(0x142, 0xa);
  STEP(0x143, 0xc);
#undef STEP
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  return wave_reduce(v, 0, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
  return wave_reduce(v, ~0u, [](uint32_t a, uint32_t b) { return min(a, b); });
}
__device__ __forceinline__ float wave_max(float v) {
  return __uint_as_float(wave_reduce(__float_as_uint(v), __float_as_uint(-INFINITY), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ __forceinline__ double wave_sum(double v) {
#define STEP(CTRL, ROWS)                                                                \
  {                                                                                     \
    const uint64_t u = __builtin_bit_cast(uint64_t, v);                                 \
    const uint32_t lo = (uint32_t)dpp_move<CTRL, ROWS>(0, (int)(uint32_t)u);            \
    const uint32_t hi = (uint32_t)dpp_move<CTRL, ROWS>(0, (int)(uint32_t)(u >> 32));    \
    v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);                           \
  }
  STEP(0x111, 0xf)
  STEP(0x112, 0xf)
  STEP(0x114, 0xf)
  STEP(0x118, 0xf)
  STEP(0x142, 0xa)
  STEP(0x143, 0xc)
#undef STEP
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// ------------------------------------------------------------------ packs
// 16 bytes of a row as stored, read at any alignment of the element.  All packs
// of a thread are read before the first is widened: a use right after its load
// would make each load wait for the one before.
struct PackBits {
  uint32_t v[4];
};

template <typename T>
struct Pack;
template <>
struct Pack<float> {
  static constexpr int N = 4;
  typedef uint32_t Raw __attribute__((ext_vector_type(4), aligned(4)));
  static __device__ __forceinline__ PackBits none() {
    return PackBits{{0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u}};
  }
  static __device__ __forceinline__ void widen(const PackBits& b, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(b.v[i]);
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<Raw*>(p) =
        Raw{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
  }
};
template <>
struct Pack<bf16> {
  static constexpr int N = 8;
  typedef uint32_t Raw __attribute__((ext_vector_type(4), aligned(2)));
  static __device__ __forceinline__ PackBits none() {
    return PackBits{{0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u}};
  }
  static __device__ __forceinline__ void widen(const PackBits& b, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(b.v[i] << 16);
      v[2 * i + 1] = __uint_as_float(b.v[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ void store(bf16* p, const float (&v)[8]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<Raw*>(p) = r;
  }
};
template <typename T>
__device__ __forceinline__ PackBits load_pack(const T* p) {
  const typename Pack<T>::Raw r = *reinterpret_cast<const typename Pack<T>::Raw*>(p);
  return PackBits{{r.x, r.y, r.z, r.w}};
}

// One pack in registers: fp32, or bf16 as stored (half the registers; each
// use widens it with one operation), which cannot hold what rules make of it.
template <typename T, bool RAW>
struct PackRegs {
  static constexpr int N = Pack<T>::N;
  float v[N];
  __device__ __forceinline__ void take(const PackBits& b) { Pack<T>::widen(b, v); }
  __device__ __forceinline__ float get(int e) const { return v[e]; }
  __device__ __forceinline__ void set(int e, float x) { v[e] = x; }
  // Elements whose bit is 0, or is set, become -inf: a bit stretched over the
  // word selects.
  __device__ __forceinline__ void keep(unsigned bits) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const uint32_t m = (uint32_t)((int)(bits << (31 - e)) >> 31);
      v[e] = __uint_as_float((__float_as_uint(v[e]) & m) | (0xFF800000u & ~m));
    }
  }
  __device__ __forceinline__ void drop(unsigned bits) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const uint32_t m = (uint32_t)((int)(bits << (31 - e)) >> 31);
      v[e] = __uint_as_float((__float_as_uint(v[e]) & ~m) | (0xFF800000u & m));
    }
  }
  __device__ __forceinline__ void clear(int e) { v[e] = -INFINITY; }
  template <int AT = 0>
  __device__ __forceinline__ void forget() {}
};
template <>
struct PackRegs<bf16, true> {
  static constexpr int N = 8;
  uint32_t v[4];
  __device__ __forceinline__ void take(const PackBits& b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = b.v[i];
  }
  __device__ __forceinline__ float get(int e) const {
    return __uint_as_float(e & 1 ? v[e >> 1] & 0xFFFF0000u : v[e >> 1] << 16);
  }
  __device__ __forceinline__ void drop(unsigned bits) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = (uint32_t)((int)(bits << (31 - 2 * i)) >> 31), hi = (uint32_t)((int)(bits << (30 - 2 * i)) >> 31);
      const uint32_t m = (lo & 0xFFFFu) | hi << 16;
      v[i] = (v[i] & ~m) | (0xFF80FF80u & m);
    }
  }
  // Widened values are not kept past here: twice the registers would be live.
  // (AT tells two branches apart, whose beginnings would be joined.)
  template <int AT = 0>
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("; %1" : "+v"(v[i]) : "n"(AT));
  }
};
template <typename P>
__device__ __forceinline__ float pack_max(const P& p) {
  float m = p.get(0);
#pragma unroll
  for (int e = 1; e < P::N; ++e) m = fmaxf(m, p.get(e));
  return m;
}

// ------------------------------------------------------------------- rows
// A part of a row in the registers of NT threads: PER packs each, in rounds of
// NT packs, and one class of the row's last classes % N (with part 0; -inf
// elsewhere).  Packs are numbered in the order that decides between equal
// logits: from the row's start, or from its end when `last` is set.
template <typename T, int NT, int PER, bool RAW>
struct RowPart {
  static constexpr int N = Pack<T>::N, kThreads = NT, kPer = PER, kClasses = NT * PER * N;
  PackRegs<T, RAW> pack[PER];
  float tail;
  template <int AT = 0>
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int j = 0; j < PER; ++j) pack[j].template forget<AT>();
  }
};
template <int N>
struct RowShape {
  int classes, full, last;
  __device__ __forceinline__ RowShape(int classes, int last) : classes(classes), full(classes / N), last(last) {}
  __device__ __forceinline__ int pack_class(int i) const { return (last ? full - 1 - i : i) * N; }
  __device__ __forceinline__ int tail_class() const { return full * N + (int)threadIdx.x; }
  __device__ __forceinline__ bool has_tail() const { return tail_class() < classes; }
  // Places in the order: packs, and the single classes behind or before them.
  __device__ __forceinline__ int pack_place(int i) const { return i + N; }
  __device__ __forceinline__ int tail_place() const {
    return last ? classes - 1 - tail_class() : full + N + (int)threadIdx.x;
  }
};

// Reads part `seg`; classes past the row are -inf, and so are packs without a
// bit in `bits` (PER of them, or null), which are not read.
template <typename P, typename T, int N>
__device__ __forceinline__ void load_part(P& d, const T* x, const RowShape<N>& s, int seg,
                                          const unsigned* bits = nullptr) {
  PackBits b[P::kPer];
#pragma unroll
  for (int j = 0; j < P::kPer; ++j) {
    const int i = (seg * P::kPer + j) * P::kThreads + (int)threadIdx.x;
    b[j] = Pack<T>::none();
    if (bits ? bits[j] != 0 : i < s.full) b[j] = load_pack(x + s.pack_class(i));
  }
  d.tail = seg == 0 && s.has_tail() ? ld1<T>(x + s.tail_class()) : -INFINITY;
#pragma unroll
  for (int j = 0; j < P::kPer; ++j) d.pack[j].take(b[j]);
}

// exp((x - m) / tau) for many x: 2^(x c - b) with c = log2(e) / tau and b = m c
// rounded, one fused operation and the hardware exponential.  What b's rounding
// leaves out, the same factor of every term, is `fix` (within 3% of one): sums
// and products take it once.  A reference so large that b would have no fraction
// left (rows at a type's lowest value, infinities) goes by the difference.
struct ExpFrom {
  float m, c, b, fix;
  bool far;
  __device__ __forceinline__ ExpFrom(float m, float c) : m(m), c(c), b(m * c) {
    far = !(fabsf(b) < 1048576.0f);
    fix = far ? 1.0f : __builtin_amdgcn_exp2f(-fmaf(m, c, -b));
  }
  template <bool FAR>
  __device__ __forceinline__ float term(float x) const {
    return __builtin_amdgcn_exp2f(FAR ? (x - m) * c : fmaf(x, c, -b));
  }
};

// Sum of the terms of a part (without `fix`).
template <bool FAR, typename P>
__device__ __forceinline__ float part_terms(P& d, const ExpFrom& from) {
  d.template forget<FAR>();
  float s = from.term<FAR>(d.tail);
#pragma unroll
  for (int j = 0; j < P::kPer; ++j)
#pragma unroll
    for (int e = 0; e < P::N; ++e) s += from.term<FAR>(d.pack[j].get(e));
  return s;
}
// The wave's sum of exp((x - m) / tau) over a part.
template <typename P>
__device__ __forceinline__ double part_sum(P& d, float m, float c) {
  const ExpFrom from(m, c);
  const float s = from.far ? part_terms<true>(d, from) : part_terms<false>(d, from);
  return wave_sum((double)s) * (double)from.fix;
}
template <typename P>
__device__ __forceinline__ float part_max(const P& d) {
  float m = d.tail;
#pragma unroll
  for (int j = 0; j < P::kPer; ++j) m = fmaxf(m, pack_max(d.pack[j]));
  return wave_max(m);
}

// Sums of exp((x - m) * c) with a reference m each, joined: (m, s) becomes the
// sum of both.  A reference of -inf has no terms.
__device__ __forceinline__ void join_sums(float& m, double& s, float om, double os, float c) {
  const float nm = fmaxf(m, om);
  if (nm == -INFINITY) return;
  s = (m == -INFINITY ? 0.0 : s * (double)__builtin_amdgcn_exp2f((m - nm) * c)) +
      (om == -INFINITY ? 0.0 : os * (double)__builtin_amdgcn_exp2f((om - nm) * c));
  m = nm;
}

// ------------------------------------------------------------------ rules
// A row of a rule table: the index given for the row, or table 0 of one, or the
// row's own.  -1 outside the table: no rule.
__device__ __forceinline__ int64_t table_row(const int32_t* index, int64_t n, int64_t row) {
  const int64_t i = index ? (int64_t)index[row] : (n == 1 ? 0 : row);
  return i >= 0 && i < n ? i : -1;
}

// One row's rules, in registers.
struct RowRules {
  const float* bias;
  const uint32_t* mask;
  const int32_t* history;
  int n_history;
  float repetition, frequency, presence;
};

__device__ __forceinline__ RowRules row_rules(const RuleParams& p, int64_t row, int classes) {
  RowRules r;
  r.bias = nullptr;
  if (p.bias) {
    const int64_t i = table_row(p.row_bias, p.n_bias, row);
    if (i >= 0) r.bias = p.bias + i * classes;
  }
  r.mask = nullptr;
  if (p.masks) {
    const int64_t i = table_row(p.row_mask, p.n_masks, row);
    if (i >= 0) r.mask = p.masks + i * ((classes + 31) / 32);
  }
  r.history = nullptr;
  r.n_history = 0;
  r.repetition = 1.0f, r.frequency = 0.0f, r.presence = 0.0f;
  if (p.history) {
    // Offsets come from device memory: kept inside the history.
    const int64_t lo = min(max(p.offsets[row], (int64_t)0), p.history_len);
    const int64_t hi = min(max(p.offsets[row + 1], lo), p.history_len);
    r.history = p.history + lo;
    r.n_history = (int)min(hi - lo, (int64_t)INT32_MAX);
    if (p.repetition) r.repetition = p.repetition[row];
    if (p.frequency) r.frequency = p.frequency[row];
    if (p.presence) r.presence = p.presence[row];
  }
  return r;
}

// The penalties of a class that stands n > 0 times in the history, every step
// rounded to fp32 by itself.
__device__ __forceinline__ float penalise(const RowRules& r, float x, int n) {
#pragma clang fp contract(off)
  x = x > 0.0f ? x / r.repetition : x * r.repetition;
  const float f = r.frequency * (float)n;
  return x - (f + r.presence);
}
// Allowed classes c .. c + N - 1 (c a multiple of N) as N bits.
template <int N>
__device__ __forceinline__ unsigned mask_bits(const uint32_t* mask, int c) {
  const unsigned b = reinterpret_cast<const uint8_t*>(mask)[c >> 3];
  return N == 8 ? b : (b >> (c & 4)) & 15u;
}
__device__ __forceinline__ bool mask_bit(const uint32_t* mask, int c) { return mask[c >> 5] >> (c & 31) & 1; }
// N biases from a table's row.
template <int N>
__device__ __forceinline__ void load_bias(const float* p, float (&v)[N]) {
#pragma unroll
  for (int q = 0; q < N; q += 4) {
    float b[4];
    Pack<float>::widen(load_pack(p + q), b);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[q + e] = b[e];
  }
}
__device__ __forceinline__ float apply_rules(const RowRules& r, float x, int c, int n) {
  if (n > 0) x = penalise(r, x, n);
  if (r.bias) x = x + r.bias[c];
  return r.mask && !mask_bit(r.mask, c) ? -INFINITY : x;
}

// Counts of the classes [first, first + n) in the row's history.
__device__ __forceinline__ void count_history(const RowRules& r, int first, int n, int* counts) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) counts[i] = 0;
  __syncthreads();
  // Four entries a thread are on their way at once.
  for (unsigned i = threadIdx.x; i < (unsigned)r.n_history; i += 4 * blockDim.x) {
    int c[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const unsigned at = i + q * blockDim.x;
      c[q] = at < (unsigned)r.n_history ? r.history[at] : -1;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (c[q] >= first && c[q] < first + n) atomicAdd(&counts[c[q] - first], 1);
  }
  __syncthreads();
}

}  // namespace ppocr
