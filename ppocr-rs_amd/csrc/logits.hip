// Operators on rows of class logits: rules (penalties, biases, masks), the
// best classes of each row, and distillation from a teacher's best classes.
#include <algorithm>
#include <cfloat>

#include "device_math.h"
#include "logits.h"

namespace ppocr {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

// Rows of a rule table: the row's own index, or table 0 of one, or its row.
// -1 outside the table: no rule.
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

// Counts of the classes [first, first + n) in the row's history.
__device__ __forceinline__ void count_history(const RowRules& r, int first, int n, int* counts) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) counts[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < r.n_history; i += blockDim.x) {
    const int c = r.history[i] - first;
    if (c >= 0 && c < n) atomicAdd(&counts[c], 1);
  }
  __syncthreads();
}

// 16 bytes of a row: its elements as fp32, at any alignment of the element.
template <typename T>
struct Pack;
template <>
struct Pack<float> {
  static constexpr int N = 4;
  typedef float Raw __attribute__((ext_vector_type(4), aligned(4)));
  static __device__ __forceinline__ void load(const float* p, float (&v)[4]) {
    const Raw r = *reinterpret_cast<const Raw*>(p);
    v[0] = r.x, v[1] = r.y, v[2] = r.z, v[3] = r.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<Raw*>(p) = Raw{v[0], v[1], v[2], v[3]};
  }
};
template <>
struct Pack<bf16> {
  static constexpr int N = 8;
  typedef uint32_t Raw __attribute__((ext_vector_type(4), aligned(2)));
  static __device__ __forceinline__ void load(const bf16* p, float (&v)[8]) {
    const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(r[i] << 16);
      v[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ void store(bf16* p, const float (&v)[8]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<Raw*>(p) = r;
  }
};

// The steps of the rules on one logit, every one rounded to fp32 by itself.
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

__device__ __forceinline__ float apply_rules(const RowRules& r, float x, int c, int n) {
  if (n > 0) x = penalise(r, x, n);
  if (r.bias) x = x + r.bias[c];
  return r.mask && !mask_bit(r.mask, c) ? -INFINITY : x;
}

// Rules of a chunk of one row: 16 elements a thread, each read and written
// once, bound by HBM.  A pack without an allowed class is not read, and in
// place one that no rule changes is neither read nor written.  Counts of the
// history's classes in the chunk are an LDS histogram, so a chunk costs one
// pass over the row's history (from L2 after the first chunk).
constexpr int kChunk = 4096;

template <typename T, bool HISTORY>
__global__ __launch_bounds__(kThreads) void logit_rules_kernel(LogitRows in, RuleParams p, T* out, int64_t out_stride,
                                                               int chunk) {
  constexpr int N = Pack<T>::N, PER = kChunk / (kThreads * N);
  __shared__ int counts[HISTORY ? kChunk : 1];
  const int64_t row = blockIdx.x;
  const int first = blockIdx.y * chunk, n = min(chunk, in.classes - first), tid = threadIdx.x;
  const RowRules r = row_rules(p, row, in.classes);
  const bool counted = HISTORY && r.n_history > 0;
  const T* x = static_cast<const T*>(in.x) + row * in.stride + first;
  T* y = out + row * out_stride + first;
  const bool in_place = x == y && !r.bias;
  const int full = n / N;
  unsigned bits[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = tid + j * kThreads;
    bits[j] = (1u << N) - 1;
    if (r.mask && i < full) bits[j] = mask_bits<N>(r.mask, first + i * N);
  }
  if (counted) count_history(r, first, n, counts);
  float v[PER][N];
  bool write[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = tid + j * kThreads;
    write[j] = i < full;
#pragma unroll
    for (int e = 0; e < N; ++e) v[j][e] = -INFINITY;
    if (write[j] && in_place && bits[j] == (1u << N) - 1) {
      write[j] = false;
      if (counted)
#pragma unroll
        for (int e = 0; e < N; ++e) write[j] |= counts[i * N + e] > 0;
    }
    if (write[j] && bits[j]) Pack<T>::load(x + i * N, v[j]);
  }
  if (counted)
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = tid + j * kThreads;
      if (write[j] && bits[j])
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int c = counts[i * N + e];
          if (c > 0) v[j][e] = penalise(r, v[j][e], c);
        }
    }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = tid + j * kThreads;
    if (!write[j]) continue;
    if (r.bias && bits[j]) {
      float b[N];
      if constexpr (N == 4) {
        Pack<float>::load(r.bias + first + i * N, b);
      } else {
        float lo[4], hi[4];
        Pack<float>::load(r.bias + first + i * N, lo);
        Pack<float>::load(r.bias + first + i * N + 4, hi);
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = lo[e], b[4 + e] = hi[e];
      }
#pragma unroll
      for (int e = 0; e < N; ++e) v[j][e] = v[j][e] + b[e];
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (!(bits[j] >> e & 1)) v[j][e] = -INFINITY;
    Pack<T>::store(y + i * N, v[j]);
  }
  // The last n % N classes, one a thread.
  if (tid < n - full * N) {
    const int i = full * N + tid;
    st1<T>(y + i, apply_rules(r, ld1<T>(x + i), first + i, counted ? counts[i] : 0));
  }
}

// A total order of (logit, class): larger is better.  NaN above all, -0 as +0,
// equal logits by class.
__device__ __forceinline__ uint64_t order_key(float x, int c, int last_ties) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  if (x != x) k = 0xFFFFFFFEu;  // below the key of all ones, which no class has
  return (uint64_t)k << 32 | (uint32_t)(last_ties ? c : ~c);
}
__device__ __forceinline__ int key_class(uint64_t k, int last_ties) { return (int)(last_ties ? (uint32_t)k : ~(uint32_t)k); }
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t h = (uint32_t)(k >> 32);
  return __uint_as_float(h & 0x80000000u ? h ^ 0x80000000u : ~h);
}
// Keys at or below this one hold -inf (no candidate).
constexpr uint64_t kNoKey = 0x007FFFFFFFFFFFFFull;

template <typename V>
__device__ __forceinline__ V block_max(V v, V* red) {
  for (int o = 32; o > 0; o >>= 1) v = max(v, (V)__shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  V r = red[0];
  for (int i = 1; i < (int)(blockDim.x >> 6); ++i) r = max(r, red[i]);
  return r;
}
__device__ __forceinline__ double block_sum(double v, double* red) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double r = red[0];
  for (int i = 1; i < (int)(blockDim.x >> 6); ++i) r += red[i];
  return r;
}

// k passes, each finding the best key below the last one.
template <typename T>
__global__ __launch_bounds__(kThreads) void top_logits_kernel(LogitRows in, TopParams p) {
  extern __shared__ int counts[];
  __shared__ uint64_t red64[16];
  __shared__ double redd[16];
  __shared__ float redf[16];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(in.x) + row * in.stride;
  const RowRules r = row_rules(p.rules, row, in.classes);
  constexpr int kSeg = 8192;
  uint64_t last = ~0ull;
  uint64_t found[kMaxTop];
  for (int j = 0; j < p.k; ++j) {
    uint64_t best = 0;
    for (int first = 0; first < in.classes; first += kSeg) {
      const int n = min(kSeg, in.classes - first);
      if (r.n_history) count_history(r, first, n, counts);
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const float v = apply_rules(r, ld1<T>(x + first + i), first + i, r.n_history ? counts[i] : 0);
        const uint64_t key = order_key(v, first + i, p.last_ties);
        if (key < last) best = max(best, key);
      }
      __syncthreads();
    }
    last = block_max(best, red64);
    found[j] = last;
    if (threadIdx.x == 0 && p.values) {
      p.values[row * p.k + j] = last > kNoKey ? key_value(last) : -INFINITY;
      p.indices[row * p.k + j] = last > kNoKey ? key_class(last, p.last_ties) : -1;
    }
  }
  // Log-sum-exp of the others, relative to their own maximum.
  const float c = kLog2e / p.temperature;
  float m = -FLT_MAX;
  double sum = 0.0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int first = 0; first < in.classes; first += kSeg) {
      const int n = min(kSeg, in.classes - first);
      if (r.n_history) count_history(r, first, n, counts);
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const float v = apply_rules(r, ld1<T>(x + first + i), first + i, r.n_history ? counts[i] : 0);
        if (order_key(v, first + i, p.last_ties) >= last) continue;
        if (pass == 0)
          m = fmaxf(m, v);
        else
          sum += (double)__builtin_amdgcn_exp2f((v - m) * c);
      }
      __syncthreads();
    }
    if (pass == 0) m = fminf(block_max(m, redf), FLT_MAX);
  }
  sum = block_sum(sum, redd);
  if (threadIdx.x != 0) return;
  const double rest = sum > 0.0 || sum != sum ? log(sum) + (double)m / p.temperature : -INFINITY;
  if (p.rest) p.rest[row] = (float)rest;
  if (p.pairs) {
    double top = 0.0;
    const float v0 = key_value(found[0]);
    for (int j = 0; j < p.k; ++j)
      if (found[j] > kNoKey) top += exp(((double)key_value(found[j]) - v0) / p.temperature);
    const double whole = top + exp(rest - (double)v0 / p.temperature);
    for (int j = 0; j < p.k; ++j) {
      const bool any = found[j] > kNoKey;
      p.pairs[(row * p.k + j) * 2] = any ? (float)key_class(found[j], p.last_ties) : -1.0f;
      p.pairs[(row * p.k + j) * 2 + 1] =
          any ? (float)(exp(((double)key_value(found[j]) - v0) / p.temperature) / whole) : 0.0f;
    }
  }
}

// The teacher's shares of one row, by one wave (k <= 64: one entry a lane).
struct TeacherRow {
  bool valid;    // this lane's entry counts
  bool any;      // some lane's does
  int index;     // its class
  double q;      // its share
  double logq;
  double q0, logq0;  // the rest's
};

__device__ __forceinline__ double wave_sum(double v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

__device__ __forceinline__ TeacherRow teacher_row(const DistillParams& p, int64_t row, int classes) {
  const int lane = threadIdx.x & 63;
  TeacherRow t;
  t.index = -1;
  float v = -INFINITY;
  if (lane < p.k) {
    t.index = p.indices[row * p.k + lane];
    v = p.values[row * p.k + lane];
  }
  t.valid = t.index >= 0 && t.index < classes && v != -INFINITY;
  if (!t.valid) t.index = -1;
  // A class named twice counts once, with its first entry.
  for (int j = 0; j < p.k; ++j) {
    const int other = __shfl(t.index, j);
    if (j < lane && other == t.index) t.valid = false;
  }
  t.any = __any(t.valid);
  if (!t.any) return t;
  const double inv = 1.0 / (double)p.temperature;
  const double d = t.valid ? (double)v * inv : -INFINITY;
  const double rest = p.rest ? (double)p.rest[row] : -INFINITY;
  const double m = fmax((double)wave_max(t.valid ? v : -INFINITY) * inv, rest);
  const double sum = wave_sum(t.valid ? exp(d - m) : 0.0) + exp(rest - m);
  const double logsum = log(sum);
  t.logq = d - m - logsum;
  t.q = t.valid ? exp(t.logq) : 0.0;
  t.logq0 = rest - m - logsum;
  t.q0 = exp(t.logq0);
  return t;
}

// Gradient of the row from its sums: classes of the rest, then the entries.
template <typename T>
__device__ __forceinline__ void distill_row_grad(const LogitRows& s, const DistillParams& p, int64_t row, float m,
                                                 float z, float mr, float zr, const TeacherRow& t, float entry) {
  const T* x = static_cast<const T*>(s.x) + row * s.stride;
  T* g = static_cast<T*>(p.grad) + row * p.grad_stride;
  const float scale = (p.grad_loss ? p.grad_loss[row] : 1.0f) * p.temperature;
  const float c = kLog2e / p.temperature;
  const bool dead = m == -INFINITY;
  const float share = zr > 0.0f ? (float)(t.q0 * exp(((double)m - mr) / p.temperature) * z / zr) : 0.0f;
  const float k = dead ? 0.0f : scale * (1.0f - share) / z;
  for (int i = threadIdx.x; i < s.classes; i += kThreads) {
    const float v = ld1<T>(x + i);
    st1<T>(g + i, dead ? 0.0f : k * __builtin_amdgcn_exp2f((v - m) * c));
  }
  __syncthreads();
  if (threadIdx.x < 64 && t.valid)
    st1<T>(g + t.index, dead ? 0.0f : scale * (__builtin_amdgcn_exp2f((entry - m) * c) / z - (float)t.q));
}

template <typename T>
__device__ __forceinline__ void zero_row(T* g, int n) {
  for (int i = threadIdx.x; i < n; i += kThreads) st1<T>(g + i, 0.0f);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_kernel(LogitRows s, DistillParams p) {
  extern __shared__ uint32_t bits[];
  __shared__ double redd[16];
  __shared__ float redf[16];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(s.x) + row * s.stride;
  const TeacherRow t = teacher_row(p, row, s.classes);
  if (!t.any) {
    if (threadIdx.x == 0) {
      if (p.loss) p.loss[row] = 0.0f;
      if (p.state)
        for (int i = 0; i < 4; ++i) p.state[row * 4 + i] = 0.0f;
    }
    if (p.grad) zero_row<T>(static_cast<T*>(p.grad) + row * p.grad_stride, s.classes);
    return;
  }
  const int words = (s.classes + 31) / 32;
  for (int i = threadIdx.x; i < words; i += kThreads) bits[i] = 0;
  __syncthreads();
  float entry = 0.0f;
  if (threadIdx.x < 64 && t.valid) {
    atomicOr(&bits[t.index >> 5], 1u << (t.index & 31));
    entry = ld1<T>(x + t.index);
  }
  __syncthreads();
  const float c = kLog2e / p.temperature;
  const double inv = 1.0 / (double)p.temperature;
  float mr = -INFINITY;
  for (int i = threadIdx.x; i < s.classes; i += kThreads)
    if (!(bits[i >> 5] >> (i & 31) & 1)) mr = fmaxf(mr, ld1<T>(x + i));
  mr = block_max(mr, redf);
  const float low = fmaxf(mr, -FLT_MAX);
  double sum = 0.0;
  for (int i = threadIdx.x; i < s.classes; i += kThreads)
    if (!(bits[i >> 5] >> (i & 31) & 1)) sum += (double)__builtin_amdgcn_exp2f((ld1<T>(x + i) - low) * c);
  const double zr = block_sum(sum, redd);
  const float m = block_max(threadIdx.x < 64 && t.valid ? fmaxf(entry, mr) : mr, redf);
  const float mlow = fmaxf(m, -FLT_MAX);
  // The whole is the entries and the rest: shares add up to one, and an error
  // of the rest's sum cancels to first order in the loss.
  const double e = threadIdx.x < 64 && t.valid ? exp(((double)entry - mlow) * inv) : 0.0;
  const double z = block_sum(e, redd) + zr * exp(((double)low - mlow) * inv);
  double term = 0.0;
  const double logz = log(z);
  if (threadIdx.x < 64 && t.valid && t.q > 0.0) term = t.q * (t.logq - (((double)entry - mlow) * inv - logz));
  if (threadIdx.x == 0 && t.q0 > 0.0) term += t.q0 * (t.logq0 - (((double)low - mlow) * inv + log(zr) - logz));
  const double loss = block_sum(term, redd) * (double)p.temperature * (double)p.temperature;
  if (threadIdx.x == 0) {
    if (p.loss) p.loss[row] = m == -INFINITY ? INFINITY : (float)loss;
    if (p.state) {
      p.state[row * 4 + 0] = m;
      p.state[row * 4 + 1] = (float)z;
      p.state[row * 4 + 2] = mr;
      p.state[row * 4 + 3] = (float)zr;
    }
  }
  if (p.grad) distill_row_grad<T>(s, p, row, m, (float)z, mr, (float)zr, t, entry);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_grad_kernel(LogitRows s, DistillParams p) {
  const int64_t row = blockIdx.x;
  const TeacherRow t = teacher_row(p, row, s.classes);
  if (!t.any) {
    zero_row<T>(static_cast<T*>(p.grad) + row * p.grad_stride, s.classes);
    return;
  }
  float entry = 0.0f;
  if (threadIdx.x < 64 && t.valid) entry = ld1<T>(static_cast<const T*>(s.x) + row * s.stride + t.index);
  __syncthreads();
  const float* st = p.state + row * 4;
  distill_row_grad<T>(s, p, row, st[0], st[1], st[2], st[3], t, entry);
}

}  // namespace

void launch_logit_rules(const LogitRows& in, const RuleParams& rules, void* out, int64_t out_stride, hipStream_t s) {
  // Chunks of equal length (whole packs), at most kChunk classes.
  const int n = (in.classes + kChunk - 1) / kChunk;
  const int chunk = ((in.classes + n - 1) / n + 7) / 8 * 8;
  const dim3 grid((unsigned)in.rows, (unsigned)((in.classes + chunk - 1) / chunk));
#define RULES_LAUNCH(T, H)                                                                                          \
  hipLaunchKernelGGL((logit_rules_kernel<T, H>), grid, dim3(kThreads), 0, s, in, rules, static_cast<T*>(out), \
                     out_stride, chunk)
  if (in.dt == DT_BF16) {
    if (rules.history)
      RULES_LAUNCH(bf16, true);
    else
      RULES_LAUNCH(bf16, false);
  } else {
    if (rules.history)
      RULES_LAUNCH(float, true);
    else
      RULES_LAUNCH(float, false);
  }
#undef RULES_LAUNCH
}

void launch_top_logits(const LogitRows& in, const TopParams& p, hipStream_t s) {
  const dim3 grid((unsigned)in.rows);
  const size_t lds = p.rules.history ? (size_t)std::min(in.classes, 8192) * sizeof(int) : 0;
  if (in.dt == DT_BF16)
    hipLaunchKernelGGL(top_logits_kernel<bf16>, grid, dim3(kThreads), lds, s, in, p);
  else
    hipLaunchKernelGGL(top_logits_kernel<float>, grid, dim3(kThreads), lds, s, in, p);
}

void launch_distill(const LogitRows& student, const DistillParams& p, hipStream_t s) {
  const dim3 grid((unsigned)student.rows);
  const size_t lds = (size_t)((student.classes + 31) / 32) * sizeof(uint32_t);
  if (student.dt == DT_BF16)
    hipLaunchKernelGGL(distill_kernel<bf16>, grid, dim3(kThreads), lds, s, student, p);
  else
    hipLaunchKernelGGL(distill_kernel<float>, grid, dim3(kThreads), lds, s, student, p);
}

void launch_distill_grad(const LogitRows& student, const DistillParams& p, hipStream_t s) {
  const dim3 grid((unsigned)student.rows);
  if (student.dt == DT_BF16)
    hipLaunchKernelGGL(distill_grad_kernel<bf16>, grid, dim3(kThreads), 0, s, student, p);
  else
    hipLaunchKernelGGL(distill_grad_kernel<float>, grid, dim3(kThreads), 0, s, student, p);
}

}  // namespace ppocr
