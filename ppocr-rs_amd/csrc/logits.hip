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
__device__ __forceinline__ double wave_sum(double v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
  return v;
}

// A part of a row in registers: PER packs a thread, pack j of thread t at
// class first + (j * NT + t) * N, and one class of the row's last
// classes % N (held with the first part; -inf elsewhere).
template <typename T, int NT, int PER>
struct RowPart {
  static constexpr int N = Pack<T>::N;
  static constexpr int kClasses = NT * PER * N;
  float v[PER][N];
  float tail;
};

// Reads part `seg` of a row, classes past the row -inf.
template <typename T, int NT, int PER>
__device__ __forceinline__ void load_part(RowPart<T, NT, PER>& d, const T* x, int classes, int seg) {
  constexpr int N = Pack<T>::N;
  const int full = classes / N;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = (seg * PER + j) * NT + (int)threadIdx.x;
    if (i < full)
      Pack<T>::load(x + i * N, d.v[j]);
    else
#pragma unroll
      for (int e = 0; e < N; ++e) d.v[j][e] = -INFINITY;
  }
  d.tail = -INFINITY;
  if (seg == 0 && (int)threadIdx.x < classes - full * N) d.tail = ld1<T>(x + full * N + threadIdx.x);
}

// The rules on a part in registers.  The history is counted in windows of
// kWindow classes, whole rounds of packs.
constexpr int kWindow = 8192;

template <typename T, int NT, int PER>
__device__ __forceinline__ void rule_part(RowPart<T, NT, PER>& d, const RowRules& r, int classes, int seg, int* counts) {
  constexpr int N = Pack<T>::N, kRounds = kWindow / (NT * N);
  static_assert(kRounds >= 1 && kWindow % (NT * N) == 0, "a window is whole rounds");
  const int full = classes / N, tail = full * N + (int)threadIdx.x;
  if (r.n_history) {
    int tail_count = 0;
#pragma unroll
    for (int w = 0; w < PER; w += kRounds) {
      const int first = (seg * PER + w) * NT * N;
      if (first >= classes) break;
      __syncthreads();  // the window before is no longer read
      count_history(r, first, min(kWindow, classes - first), counts);
      if (tail >= first && tail < min(first + kWindow, classes)) tail_count = counts[tail - first];
#pragma unroll
      for (int j = w; j < w + kRounds && j < PER; ++j) {
        const int i = (seg * PER + j) * NT + (int)threadIdx.x;
        if (i < full)
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const int c = counts[i * N + e - first];
            if (c > 0) d.v[j][e] = penalise(r, d.v[j][e], c);
          }
      }
    }
    // The row's last classes may lie in a window behind their part.
    if (seg == 0 && tail < classes) {
      if (tail >= PER * NT * N)
        for (int i = 0; i < r.n_history; ++i) tail_count += r.history[i] == tail;
      if (tail_count > 0) d.tail = penalise(r, d.tail, tail_count);
    }
  }
  if (r.bias) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = (seg * PER + j) * NT + (int)threadIdx.x;
      if (i < full)
#pragma unroll
        for (int q = 0; q < N; q += 4) {
          float b[4];
          Pack<float>::load(r.bias + i * N + q, b);
#pragma unroll
          for (int e = 0; e < 4; ++e) d.v[j][q + e] = d.v[j][q + e] + b[e];
        }
    }
    if (seg == 0 && tail < classes) d.tail = d.tail + r.bias[tail];
  }
  if (r.mask) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = (seg * PER + j) * NT + (int)threadIdx.x;
      const unsigned bits = i < full ? mask_bits<N>(r.mask, i * N) : 0;
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (!(bits >> e & 1)) d.v[j][e] = -INFINITY;
    }
    if (seg == 0 && tail < classes && !mask_bit(r.mask, tail)) d.tail = -INFINITY;
  }
}

template <typename T, int NT, int PER, bool RULES>
__device__ __forceinline__ void read_part(RowPart<T, NT, PER>& d, const T* x, const RowRules& r, int classes, int seg,
                                          int* counts) {
  load_part(d, x, classes, seg);
  if constexpr (RULES) rule_part(d, r, classes, seg, counts);
}

template <int N>
__device__ __forceinline__ float pack_max(const float (&v)[N]) {
  float m = v[0];
#pragma unroll
  for (int e = 1; e < N; ++e) m = fmaxf(m, v[e]);
  return m;
}

// Wave sums of exp((x - max) * c) with their own maxima, joined over the parts
// of a row: (m, s) becomes the sum of both.  -inf is no maximum.
__device__ __forceinline__ void join_sums(float& m, double& s, float om, double os, float c) {
  const float nm = fmaxf(m, om);
  if (nm == -INFINITY) return;
  s = (m == -INFINITY ? 0.0 : s * (double)__builtin_amdgcn_exp2f((m - nm) * c)) +
      (om == -INFINITY ? 0.0 : os * (double)__builtin_amdgcn_exp2f((om - nm) * c));
  m = nm;
}

// The sum of exp((v - m) * c) over a part, m the wave's maximum of it, limited to
// finite numbers: +inf then counts as an infinite term and -inf as none.
template <typename T, int NT, int PER>
__device__ __forceinline__ void part_sum(const RowPart<T, NT, PER>& d, float c, float& m, double& sum) {
  constexpr int N = Pack<T>::N;
  float t = d.tail;
#pragma unroll
  for (int j = 0; j < PER; ++j) t = fmaxf(t, pack_max(d.v[j]));
  m = wave_max(t);
  const float ref = fminf(fmaxf(m, -FLT_MAX), FLT_MAX);
  float s = __builtin_amdgcn_exp2f((d.tail - ref) * c);
#pragma unroll
  for (int j = 0; j < PER; ++j)
#pragma unroll
    for (int e = 0; e < N; ++e) s += __builtin_amdgcn_exp2f((d.v[j][e] - ref) * c);
  sum = wave_sum((double)s);
  // A NaN is no maximum but must not be lost.
  if (m == -INFINITY && sum != sum) m = -FLT_MAX;
  m = fminf(m, FLT_MAX);
}

// The k best classes of a row and the log-sum-exp of the others, one row a
// workgroup, the row read once (parts of longer rows a second time).
//
// Every group of NT / 256 threads has its best (logit, first pack that holds
// it).  The k-th best of the 256 groups bounds the k-th best class from below,
// and only about k groups hold classes above the bound: those go to a list in
// LDS, out of the registers, and each finds its rank by counting the better
// ones.  What is left in the registers and the list's tail is the rest.  The
// bound is found by bisection over the groups' order keys, every wave for
// itself.  A list that overflows (rows whose best classes crowd in few threads)
// sends the row to k searches for the next best class.
constexpr int kGroups = 256, kList = 512;

struct TopShared {
  uint32_t group_key[kGroups], group_pack[kGroups];
  uint64_t list[kList], sorted[kList];
  uint64_t red[16];
  double wave_sum[16];
  float wave_max[16];
  int n_list;
};

// Bound of the list: the composite (key, pack) that at least k groups reach,
// and few more.
__device__ __forceinline__ uint64_t top_bound(const TopShared& sh, int k) {
  const int lane = threadIdx.x & 63;
  uint32_t key[4], pack[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) key[i] = sh.group_key[i * 64 + lane], pack[i] = sh.group_pack[i * 64 + lane];
  const auto reach = [&](uint32_t t) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) n += __popcll(__ballot(key[i] >= t));
    return n;
  };
  const uint32_t none = (uint32_t)(kNoKey >> 32);
  if (reach(none + 1) <= k) return (uint64_t)(none + 1) << 32;
  uint32_t lo = none + 1;
  uint32_t hi = wave_max(max(max(key[0], key[1]), max(key[2], key[3]))) + 1;
  // A smaller start for rows without -inf groups.
  const uint32_t low = ~wave_max(~min(min(key[0], key[1]), min(key[2], key[3])));
  lo = max(lo, low);
  int n = kGroups;
  const int enough = k + k / 2 + 8;
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    const int c = reach(mid);
    if (c >= k) {
      lo = mid;
      n = c;
      if (n <= enough) break;
    } else {
      hi = mid;
    }
  }
  if (n <= enough) return (uint64_t)lo << 32;
  // Many groups tie at the bound: the first packs among them.
  const int need = k - reach(lo + 1);
  uint32_t plo = 0, phi = 0xFFFFFFFFu;
  while (phi - plo > 1) {
    const uint32_t mid = plo + (phi - plo) / 2;
    int c = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) c += __popcll(__ballot(key[i] == lo && pack[i] >= mid));
    if (c >= need)
      plo = mid;
    else
      phi = mid;
  }
  return (uint64_t)lo << 32 | plo;
}

// The slow way for any row: k searches for the best class below the last one,
// then the sums of the others, the row read each time.
template <typename T, bool RULES>
__device__ __forceinline__ void search_row(const T* x, const RowRules& r, int classes, const TopParams& p, float c,
                                        int* counts, TopShared& sh, float& wm, double& ws) {
  const auto each = [&](auto&& f) {
    for (int first = 0; first < classes; first += kWindow) {
      const int n = min(kWindow, classes - first);
      bool counted = false;
      if constexpr (RULES) {
        counted = r.n_history > 0;
        if (counted) {
          __syncthreads();
          count_history(r, first, n, counts);
        }
      }
      for (int i = threadIdx.x; i < n; i += blockDim.x) {
        float v = ld1<T>(x + first + i);
        if constexpr (RULES) v = apply_rules(r, v, first + i, counted ? counts[i] : 0);
        f(v, order_key(v, first + i, p.last_ties));
      }
    }
  };
  uint64_t last = ~0ull;
  for (int j = 0; j < p.k; ++j) {
    uint64_t next = 0;
    each([&](float, uint64_t key) { next = key < last ? max(next, key) : next; });
    last = block_max(next, sh.red);
    if (threadIdx.x == 0) sh.sorted[j] = last;
  }
  float m = -FLT_MAX;
  bool some = false;
  each([&](float v, uint64_t key) {
    if (key < last && v != -INFINITY) some = true, m = fmaxf(m, v);
  });
  m = fminf(wave_max(m), FLT_MAX);
  double sum = 0.0;
  each([&](float v, uint64_t key) {
    if (key < last) sum += (double)__builtin_amdgcn_exp2f((v - m) * c);
  });
  wm = __any(some) ? m : -INFINITY;
  ws = wave_sum(sum);
}

template <typename T, int NT, int PER, bool RULES>
__global__ __launch_bounds__(NT, NT == 1024 ? 4 : PER * Pack<T>::N <= 32 ? 5 : RULES ? 3 : 4) void top_logits_kernel(LogitRows in, TopParams p, int segs) {
  constexpr int N = Pack<T>::N, W = NT / 64;
  __shared__ TopShared sh;
  extern __shared__ int counts[];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(in.x) + row * in.stride;
  RowRules r{};
  if constexpr (RULES) r = row_rules(p.rules, row, in.classes);
  const int tail_class = in.classes / N * N + tid;
  const float c = kLog2e / p.temperature;
  if (tid == 0) sh.n_list = 0;

  // Best logit of this thread and the first pack that holds it.
  RowPart<T, NT, PER> d;
  float best = -INFINITY;
  int pack = 0;
  bool nan = false;
  int nan_pack = 0;
  for (int seg = 0; seg < segs; ++seg) {
    read_part<T, NT, PER, RULES>(d, x, r, in.classes, seg, counts);
    bool bad = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const float m = pack_max(d.v[j]);
      const bool better = m > best || (p.last_ties && m == best);
      best = better ? m : best;
      pack = better ? ((seg * PER + j) * NT + tid) * N : pack;
#pragma unroll
      for (int e = 0; e < N; e += 2) bad |= __builtin_isunordered(d.v[j][e], d.v[j][e + 1]);
    }
    if (bad && (!nan || p.last_ties)) {
#pragma unroll
      for (int j = 0; j < PER; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (d.v[j][e] != d.v[j][e] && (!nan || p.last_ties)) nan = true, nan_pack = ((seg * PER + j) * NT + tid) * N;
    }
    if (seg == 0) {
      // The single class at the row's end comes after the thread's packs.
      if (d.tail > best || (p.last_ties && d.tail == best)) best = d.tail, pack = tail_class;
      if (d.tail != d.tail && (!nan || p.last_ties)) nan = true, nan_pack = tail_class;
    }
  }
  uint64_t mine = order_key(nan ? NAN : best, nan ? nan_pack : pack, p.last_ties);
  if constexpr (NT > kGroups) {
#pragma unroll
    for (int o = 1; o < NT / kGroups; o <<= 1) mine = max(mine, (uint64_t)__shfl_xor((unsigned long long)mine, o));
  }
  if (tid % (NT / kGroups) == 0) {
    sh.group_key[tid / (NT / kGroups)] = (uint32_t)(mine >> 32);
    sh.group_pack[tid / (NT / kGroups)] = (uint32_t)mine;
  }
  __syncthreads();

  // Classes above the bound into the list; the others' sums.
  const uint64_t bound = top_bound(sh, p.k);
  const float floor_value = key_value(bound);
  float wm = -INFINITY;
  double ws = 0.0;
  for (int seg = segs - 1; seg >= 0; --seg) {
    if (seg != segs - 1) read_part<T, NT, PER, RULES>(d, x, r, in.classes, seg, counts);
    const auto take = [&](float& v, int cls, int at) {
      const uint64_t key = order_key(v, at, p.last_ties);
      if (key < bound || key <= kNoKey) return;
      const int slot = atomicAdd(&sh.n_list, 1);
      if (slot < kList) sh.list[slot] = order_key(v, cls, p.last_ties);
      v = -INFINITY;
    };
    if (best >= floor_value || nan) {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (pack_max(d.v[j]) >= floor_value || nan) {
          const int at = ((seg * PER + j) * NT + tid) * N;
#pragma unroll
          for (int e = 0; e < N; ++e) take(d.v[j][e], at + e, at);
        }
      }
      if (seg == 0) take(d.tail, tail_class, tail_class);
    }
    float m;
    double s;
    part_sum(d, c, m, s);
    join_sums(wm, ws, m, s, c);
  }
  if (lane == 0) sh.wave_max[wave] = wm, sh.wave_sum[wave] = ws;
  __syncthreads();

  int n = sh.n_list;
  if (n <= kList) {
    for (int i = tid; i < n; i += NT) {
      const uint64_t key = sh.list[i];
      int rank = 0;
      for (int o = 0; o < n; ++o) rank += sh.list[o] > key;
      sh.sorted[rank] = key;
    }
  } else {
    search_row<T, RULES>(x, r, in.classes, p, c, counts, sh, wm, ws);
    n = p.k;
    if (lane == 0) sh.wave_max[wave] = wm, sh.wave_sum[wave] = ws;
  }
  __syncthreads();
  if (wave != 0) return;

  // The best of the list, and the rest: the list's tail and the waves' sums.
  const uint64_t key = lane < min(n, p.k) ? sh.sorted[lane] : 0;
  const bool any = key > kNoKey;
  if (p.values && lane < p.k) {
    p.values[row * p.k + lane] = any ? key_value(key) : -INFINITY;
    p.indices[row * p.k + lane] = any ? key_class(key, p.last_ties) : -1;
  }
  if (!p.rest && !p.pairs) return;
  float m = lane < W ? sh.wave_max[lane] : -INFINITY;
  for (int i = p.k + lane; i < n; i += 64) {
    const float v = key_value(sh.sorted[i]);
    m = fmaxf(m, v != v ? FLT_MAX : v);
  }
  m = fminf(wave_max(m), FLT_MAX);
  const double inv = 1.0 / (double)p.temperature;
  double sum = 0.0;
  if (lane < W && sh.wave_max[lane] > -INFINITY) sum = sh.wave_sum[lane] * exp(((double)sh.wave_max[lane] - m) * inv);
  for (int i = p.k + lane; i < n; i += 64) sum += exp(((double)key_value(sh.sorted[i]) - m) * inv);
  sum = wave_sum(sum);
  const double rest = m == -INFINITY ? -INFINITY : log(sum) + (double)m * inv;
  if (p.rest && lane == 0) p.rest[row] = (float)rest;
  if (p.pairs) {
    const double top = __shfl((double)key_value(key), 0) * inv;
    const double e = any ? exp((double)key_value(key) * inv - top) : 0.0;
    const double whole = wave_sum(e) + (m == -INFINITY ? 0.0 : exp(rest - top));
    if (lane < p.k) {
      p.pairs[(row * p.k + lane) * 2] = any ? (float)key_class(key, p.last_ties) : -1.0f;
      p.pairs[(row * p.k + lane) * 2 + 1] = any ? (float)(e / whole) : 0.0f;
    }
  }
}

// An entry of a teacher's row, one a lane (k <= 64).
struct TeacherEntry {
  int index;  // its class, -1: does not count (a class named twice is not looked for yet)
  float value;
};
__device__ __forceinline__ TeacherEntry teacher_entry(const DistillParams& p, int64_t row, int classes) {
  const int lane = threadIdx.x & 63;
  TeacherEntry t{-1, -INFINITY};
  if (lane < p.k) {
    t.index = p.indices[row * p.k + lane];
    t.value = p.values[row * p.k + lane];
  }
  if (t.index < 0 || t.index >= classes || t.value == -INFINITY) t.index = -1;
  return t;
}

// The teacher's shares of a row, by one wave, in 64 bits: the loss is a
// difference of logs that nearly cancel.
struct TeacherShares {
  bool valid;     // this lane's entry counts
  double q, logq;  // its share
  double q0, logq0;  // the rest's
};
__device__ __forceinline__ TeacherShares teacher_shares(const DistillParams& p, int64_t row, const TeacherEntry& e,
                                                        double inv) {
  const int lane = threadIdx.x & 63;
  TeacherShares t;
  t.valid = e.index >= 0;
  // A class named twice counts once, with its first entry.
  for (int j = 0; j + 1 < p.k; ++j)
    if (__builtin_amdgcn_readlane(e.index, j) == e.index && j < lane) t.valid = false;
  const double rest = p.rest ? (double)p.rest[row] : -INFINITY;
  const double m = fmax((double)wave_max(t.valid ? e.value : -INFINITY) * inv, rest);
  const double d = (double)e.value * inv - m;
  const double x = t.valid ? exp(d) : 0.0, x0 = exp(rest - m);
  const double sum = wave_sum(x) + x0, logsum = log(sum);
  t.q = x / sum;
  t.logq = d - logsum;
  t.q0 = x0 / sum;
  t.logq0 = rest - m - logsum;
  return t;
}

// Distillation of one row a workgroup: its loss, its gradient, or both.
//
// With e_c = exp((s_c - M) / tau), Z0 the sum of e over the classes that are no
// entry, Z = Z0 + sum over the entries, p = e / Z and the rest's share of the
// student p0 = Z0 / Z:
//   loss = tau^2 (sum_j q_j (log q_j - log p_j) + q0 (log q0 - log p0)),
//   d loss / d s_c = tau (p_c - q_c) for an entry, tau e_c (1 / Z - q0 / Z0) else.
// So the rest's gradient is e times one factor of the row, and the row is read
// once: it stays in registers with the entries taken out (their marks come
// through LDS, a byte a pack), first as logits, then as exponentials relative
// to the wave's maximum.  Wave 0 does the entries, in 64 bits, while the others
// sum, and writes their gradients over the row's.  The whole is formed from the
// rest and the entries, so that the shares add up to one and an error of the
// rest's sum cancels to first order in the loss.  Rows longer than the
// registers go through them in parts, twice when the gradient is asked for.
enum DistillMode { kLoss, kBoth, kGradient };

struct DistillShared {
  double sum[16];
  float max[16];
  float factor[16];
  float top;  // maximum of the rest
};

// PARTS: rows of `segs` parts; else the whole row is one.
template <typename T, int NT, int PER, bool PARTS, DistillMode MODE>
__global__ __launch_bounds__(NT, NT == 1024 ? 4 : PER * Pack<T>::N <= 32 ? 6 : 4) void distill_kernel(
    LogitRows s, DistillParams p, int parts) {
  constexpr int N = Pack<T>::N, W = NT / 64, kWords = (PER + 3) / 4;
  __shared__ DistillShared sh;
  __shared__ uint32_t marks[MODE == kGradient ? 1 : NT * kWords];
  const int segs = PARTS ? parts : 1;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const int full = s.classes / N, tail_class = full * N + tid;
  const bool has_tail = tail_class < s.classes;
  const T* x = static_cast<const T*>(s.x) + row * s.stride;
  T* g = static_cast<T*>(p.grad) + row * p.grad_stride;
  const TeacherEntry entry = teacher_entry(p, row, s.classes);
  if (!__any(entry.index >= 0)) {
    if (MODE != kGradient && tid == 0) p.loss[row] = 0.0f;
    if (MODE == kLoss && p.state && tid < 4) p.state[row * 4 + tid] = 0.0f;
    if (MODE != kLoss) {
      const float zero[N] = {};
      for (int i = tid; i < full; i += NT) Pack<T>::store(g + i * N, zero);
      if (has_tail) st1<T>(g + tail_class, 0.0f);
    }
    return;
  }
  const float c = kLog2e / p.temperature;
  const double inv = 1.0 / (double)p.temperature;
  // The entries' own logits, before a gradient in place covers them.
  float own = 0.0f;
  if (wave == 0 && entry.index >= 0) own = ld1<T>(x + entry.index);

  RowPart<T, NT, PER> d;
  float m = -INFINITY;  // the wave's maximum and sum of the rest
  double sum = 0.0;
  if constexpr (MODE != kGradient) {
    for (int seg = 0; seg < segs; ++seg) {
      load_part(d, x, s.classes, seg);
#pragma unroll
      for (int i = 0; i < kWords; ++i) marks[tid * kWords + i] = 0;
      __syncthreads();
      if (wave == 0 && entry.index >= 0) {
        const int i = entry.index / N, at = i - seg * PER * NT;
        if (i < full && at >= 0 && at < PER * NT) {
          const int j = at / NT;
          atomicOr(&marks[(at - j * NT) * kWords + (j >> 2)], 1u << ((j & 3) * 8 + entry.index % N));
        }
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        const uint32_t word = marks[tid * kWords + w];
        if (word)
#pragma unroll
          for (int q = 0; q < 4 && w * 4 + q < PER; ++q)
#pragma unroll
            for (int e = 0; e < N; ++e)
              if (word >> (q * 8 + e) & 1) d.v[w * 4 + q][e] = -INFINITY;
      }
      if (seg == 0 && __any(entry.index >= full * N)) {
        // Entries among the row's last classes, one a thread.
        for (int j = 0; j < p.k; ++j)
          if (__builtin_amdgcn_readlane(entry.index, j) == tail_class) d.tail = -INFINITY;
      }
      float t = d.tail;
#pragma unroll
      for (int j = 0; j < PER; ++j) t = fmaxf(t, pack_max(d.v[j]));
      t = wave_max(t);
      const float ref = fmaxf(t, -FLT_MAX);
      d.tail = __builtin_amdgcn_exp2f((d.tail - ref) * c);
      float part = d.tail;
#pragma unroll
      for (int j = 0; j < PER; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          d.v[j][e] = __builtin_amdgcn_exp2f((d.v[j][e] - ref) * c);
          part += d.v[j][e];
        }
      const double ps = wave_sum((double)part);
      if (ps != ps) t = ref;  // a NaN is no maximum but must not be lost
      join_sums(m, sum, t, ps, c);
      if (PARTS) __syncthreads();  // the marks are no longer read
    }
    if (lane == 0) sh.max[wave] = m, sh.sum[wave] = sum;
    __syncthreads();
  } else if (!PARTS) {
    load_part(d, x, s.classes, 0);
  }

  float entry_grad = 0.0f;
  bool entry_valid = false;
  if (wave == 0) {
    const TeacherShares t = teacher_shares(p, row, entry, inv);
    entry_valid = t.valid;
    double top, z, mr, zr;
    if constexpr (MODE == kGradient) {
      const float* st = p.state + row * 4;
      top = st[0], z = st[1], mr = st[2], zr = st[3];
    } else {
      const float om = lane < W ? sh.max[lane] : -INFINITY;
      const float rm = wave_max(om);
      // Sums of the waves; a wave without any class of the rest has none.
      zr = wave_sum(om > -INFINITY ? sh.sum[lane] * exp(((double)om - rm) * inv) : 0.0);
      mr = rm;
      const float em = fmaxf(rm, wave_max(t.valid ? own : -INFINITY));
      top = em;
    }
    const double low = fmax(top, -(double)FLT_MAX);
    const double a = ((double)own - low) * inv;
    const double e = t.valid ? exp(a) : 0.0;
    const double e0 = mr == -INFINITY ? 0.0 : exp((mr - low) * inv);  // of the rest's maximum
    if constexpr (MODE != kGradient) {
      z = wave_sum(e) + zr * e0;
      const double logz = log(z);
      double term = t.valid && t.q > 0.0 ? t.q * (t.logq - (a - logz)) : 0.0;
      if (lane == 0 && t.q0 > 0.0) term += t.q0 * (t.logq0 - (zr > 0.0 || zr != zr ? (mr - low) * inv + log(zr) - logz : -INFINITY));
      const double loss = wave_sum(term) * (double)p.temperature * (double)p.temperature;
      if (lane == 0) {
        p.loss[row] = top == -INFINITY && !(z != z) ? INFINITY : (float)loss;
        if (MODE == kLoss && p.state) {
          p.state[row * 4 + 0] = (float)top;
          p.state[row * 4 + 1] = (float)z;
          p.state[row * 4 + 2] = (float)mr;
          p.state[row * 4 + 3] = (float)zr;
        }
      }
    }
    if constexpr (MODE != kLoss) {
      const double scale = (p.grad_loss ? (double)p.grad_loss[row] : 1.0) * (double)p.temperature;
      // No class has any probability: no gradient.
      const bool dead = top == -INFINITY && !(z != z);
      // Of exponentials relative to the rest's maximum: its classes may be far
      // below the entries and still share q0 among them.
      const double factor = dead || zr == 0.0 ? 0.0 : scale * (e0 / z - t.q0 / zr);
      entry_grad = dead ? 0.0f : (float)(scale * (e / z - t.q));
      if (MODE == kBoth && !PARTS) {
        // The registers hold exponentials of each wave's own maximum.
        if (lane < W) sh.factor[lane] = sh.max[lane] == -INFINITY ? 0.0f : (float)(factor * exp(((double)sh.max[lane] - mr) * inv));
      } else if (lane == 0) {
        sh.factor[0] = (float)factor;
        sh.top = (float)fmax(mr, -(double)FLT_MAX);
      }
    }
  }
  if constexpr (MODE != kLoss) {
    __syncthreads();
    constexpr bool kReady = MODE == kBoth && !PARTS;
    const float factor = sh.factor[kReady ? wave : 0], ref = kReady ? 0.0f : sh.top;
    for (int seg = segs - 1; seg >= 0; --seg) {
      if (PARTS) load_part(d, x, s.classes, seg);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = (seg * PER + j) * NT + tid;
        if (i >= full) continue;
        float v[N];
#pragma unroll
        for (int e = 0; e < N; ++e)
          v[e] = factor * (kReady ? d.v[j][e] : __builtin_amdgcn_exp2f((d.v[j][e] - ref) * c));
        Pack<T>::store(g + i * N, v);
      }
      if (seg == 0 && has_tail)
        st1<T>(g + tail_class, factor * (kReady ? d.tail : __builtin_amdgcn_exp2f((d.tail - ref) * c)));
    }
    __syncthreads();
    if (wave == 0 && entry_valid) st1<T>(g + entry.index, entry_grad);
  }
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

template <typename T, int NT, int PER, bool RULES>
void launch_top(const LogitRows& in, const TopParams& p, hipStream_t s) {
  const int segs = (in.classes + RowPart<T, NT, PER>::kClasses - 1) / RowPart<T, NT, PER>::kClasses;
  const size_t lds = p.rules.history ? kWindow * sizeof(int) : 0;
  hipLaunchKernelGGL((top_logits_kernel<T, NT, PER, RULES>), dim3((unsigned)in.rows), dim3(NT), lds, s, in, p, segs);
}

// Threads of a row's workgroup and the elements that each holds.
template <typename T, bool RULES>
void launch_top_typed(const LogitRows& in, const TopParams& p, hipStream_t s) {
  constexpr int N = Pack<T>::N, kLong = RULES ? 64 : 80;
  if (in.rows < 512 && in.classes > 256 * 8)
    in.classes <= 1024 * 32 ? launch_top<T, 1024, 32 / N, RULES>(in, p, s)
                            : launch_top<T, 1024, kLong / N, RULES>(in, p, s);
  else if (in.classes <= 256 * 32)
    launch_top<T, 256, 32 / N, RULES>(in, p, s);
  else if (in.classes <= 256 * 80)
    launch_top<T, 256, 80 / N, RULES>(in, p, s);
  else
    launch_top<T, 1024, kLong / N, RULES>(in, p, s);
}

void launch_top_logits(const LogitRows& in, const TopParams& p, hipStream_t s) {
  if (p.rules.history || p.rules.bias || p.rules.masks)
    in.dt == DT_BF16 ? launch_top_typed<bf16, true>(in, p, s) : launch_top_typed<float, true>(in, p, s);
  else
    in.dt == DT_BF16 ? launch_top_typed<bf16, false>(in, p, s) : launch_top_typed<float, false>(in, p, s);
}

template <typename T, int NT, int PER, bool PARTS, DistillMode MODE>
void launch_distill_one(const LogitRows& in, const DistillParams& p, hipStream_t s) {
  const int parts = (in.classes + RowPart<T, NT, PER>::kClasses - 1) / RowPart<T, NT, PER>::kClasses;
  hipLaunchKernelGGL((distill_kernel<T, NT, PER, PARTS, MODE>), dim3((unsigned)in.rows), dim3(NT), 0, s, in, p, parts);
}

// Threads of a row's workgroup and the elements that each holds.
template <typename T, DistillMode MODE>
void launch_distill_typed(const LogitRows& in, const DistillParams& p, hipStream_t s) {
  constexpr int N = Pack<T>::N;
  if (in.rows < 512 && in.classes > 256 * 8 && in.classes <= 1024 * 32)
    launch_distill_one<T, 1024, 32 / N, false, MODE>(in, p, s);
  else if (in.classes <= 256 * 32)
    launch_distill_one<T, 256, 32 / N, false, MODE>(in, p, s);
  else if (in.classes <= 256 * 80)
    launch_distill_one<T, 256, 80 / N, false, MODE>(in, p, s);
  else
    launch_distill_one<T, 1024, 80 / N, true, MODE>(in, p, s);
}

template <DistillMode MODE>
void launch_distill_mode(const LogitRows& in, const DistillParams& p, hipStream_t s) {
  in.dt == DT_BF16 ? launch_distill_typed<bf16, MODE>(in, p, s) : launch_distill_typed<float, MODE>(in, p, s);
}

void launch_distill(const LogitRows& student, const DistillParams& p, hipStream_t s) {
  p.grad ? launch_distill_mode<kBoth>(student, p, s) : launch_distill_mode<kLoss>(student, p, s);
}

void launch_distill_grad(const LogitRows& student, const DistillParams& p, hipStream_t s) {
  launch_distill_mode<kGradient>(student, p, s);
}

}  // namespace ppocr
