// The best classes of rows of class logits and the log-sum-exp of the others.
#include "logit_rows.h"

namespace ppocr {
namespace {

// A total order of (logit, class): larger is better.  NaN above all, -0 as +0,
// equal logits by class.
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return x != x ? 0xFFFFFFFEu : k;  // below the key of all ones, which no class has
}
__device__ __forceinline__ uint64_t order_key(float x, int c, int last) {
  return (uint64_t)value_key(x) << 32 | (uint32_t)(last ? c : ~c);
}
__device__ __forceinline__ int key_class(uint64_t k, int last) { return (int)(last ? (uint32_t)k : ~(uint32_t)k); }
__device__ __forceinline__ float key_value(uint32_t h) {
  return __uint_as_float(h & 0x80000000u ? h ^ 0x80000000u : ~h);
}
__device__ __forceinline__ float key_value(uint64_t k) { return key_value((uint32_t)(k >> 32)); }
// Value key of -inf, which is no candidate.
constexpr uint32_t kNone = 0x007FFFFFu;
constexpr uint64_t kNoKey = (uint64_t)kNone << 32 | 0xFFFFFFFFu;

__device__ __forceinline__ uint64_t block_max(uint64_t v, uint64_t* red) {
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint64_t)__shfl_xor((unsigned long long)v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t r = red[0];
  for (int i = 1; i < (int)(blockDim.x >> 6); ++i) r = max(r, red[i]);
  return r;
}

// The rules on a part in registers.  The history is counted in windows of
// kWindow classes, whole rounds of packs; the row's last classes have counters
// of their own behind the window's.
constexpr int kWindow = 8192;

template <typename P, int N>
__device__ __forceinline__ void rule_part(P& d, const RowRules& r, const RowShape<N>& s, int seg, int* counts) {
  constexpr int NT = P::kThreads, PER = P::kPer, kRounds = kWindow / (NT * N);
  static_assert(kRounds >= 1 && kWindow % (NT * N) == 0, "a window is whole rounds");
  const int tail = s.tail_class();
  if (r.n_history) {
    if (seg == 0 && s.full * N < s.classes) {
      __syncthreads();
      count_history(r, s.full * N, s.classes - s.full * N, counts + kWindow);
      if (tail < s.classes && counts[kWindow + threadIdx.x] > 0)
        d.tail = penalise(r, d.tail, counts[kWindow + threadIdx.x]);
    }
#pragma unroll
    for (int w = 0; w < PER; w += kRounds) {
      const int i0 = (seg * PER + w) * NT, i1 = min(i0 + kRounds * NT, s.full);
      if (i0 < s.full) {
        const int first = min(s.pack_class(i0), s.pack_class(i1 - 1));
        __syncthreads();  // the window before is no longer read
        count_history(r, first, (i1 - i0) * N, counts);
#pragma unroll
        for (int j = w; j < w + kRounds && j < PER; ++j) {
          const int i = (seg * PER + j) * NT + (int)threadIdx.x;
          if (i < s.full)
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const int c = counts[s.pack_class(i) - first + e];
              if (c > 0) d.pack[j].set(e, penalise(r, d.pack[j].get(e), c));
            }
        }
      }
    }
  }
  if (r.bias) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = (seg * PER + j) * NT + (int)threadIdx.x;
      if (i < s.full) {
        float b[N];
        load_bias<N>(r.bias + s.pack_class(i), b);
#pragma unroll
        for (int e = 0; e < N; ++e) d.pack[j].set(e, d.pack[j].get(e) + b[e]);
      }
    }
    if (seg == 0 && tail < s.classes) d.tail = d.tail + r.bias[tail];
  }
  if (r.mask) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = (seg * PER + j) * NT + (int)threadIdx.x;
      const unsigned bits = i < s.full ? mask_bits<N>(r.mask, s.pack_class(i)) : 0;
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (!(bits >> e & 1)) d.pack[j].clear(e);
    }
    if (seg == 0 && tail < s.classes && !mask_bit(r.mask, tail)) d.tail = -INFINITY;
  }
}

template <bool RULES, typename P, typename T, int N>
__device__ __forceinline__ void read_part(P& d, const T* x, const RowRules& r, const RowShape<N>& s, int seg, int* counts) {
  load_part(d, x, s, seg);
  if constexpr (RULES) rule_part(d, r, s, seg, counts);
}

// Sums of exp((x - max) * c) with their own maxima, joined: (m, s) becomes the
// sum of both.  -inf is no maximum.
__device__ __forceinline__ void join_sums(float& m, double& s, float om, double os, float c) {
  const float nm = fmaxf(m, om);
  if (nm == -INFINITY) return;
  s = (m == -INFINITY ? 0.0 : s * (double)__builtin_amdgcn_exp2f((m - nm) * c)) +
      (om == -INFINITY ? 0.0 : os * (double)__builtin_amdgcn_exp2f((om - nm) * c));
  m = nm;
}

// The sum of exp((v - m) * c) over a part, m the wave's maximum of it, limited to
// finite numbers: +inf then counts as an infinite term and -inf as none.
template <typename P>
__device__ __forceinline__ void part_sum(P& d, float c, float& m, double& sum) {
  float t = d.tail;
#pragma unroll
  for (int j = 0; j < P::kPer; ++j) t = fmaxf(t, pack_max(d.pack[j]));
  m = wave_max(t);
  d.forget();
  const float ref = fminf(fmaxf(m, -FLT_MAX), FLT_MAX);
  float s = __builtin_amdgcn_exp2f((d.tail - ref) * c);
#pragma unroll
  for (int j = 0; j < P::kPer; ++j)
#pragma unroll
    for (int e = 0; e < P::N; ++e) s += __builtin_amdgcn_exp2f((d.pack[j].get(e) - ref) * c);
  sum = wave_sum((double)s);
  // A NaN is no maximum but must not be lost.
  if (m == -INFINITY && sum != sum) m = -FLT_MAX;
  m = fminf(m, FLT_MAX);
}

// The k best classes of a row and the log-sum-exp of the others, one row a
// workgroup, the row read once (parts of longer rows a second time).
//
// Every group of NT / 256 threads has its best (logit, first place that holds
// it).  The k-th best of the 256 groups bounds the k-th best class from below,
// and only about k groups hold classes above the bound: those go to a list in
// LDS, out of the registers, and each finds its rank by counting the better
// ones.  What is left in the registers and the list's end is the rest.  The
// bound is found by bisection over the groups' order keys, every wave for
// itself.  A list that overflows (rows whose best classes crowd in few threads)
// sends the row to k searches for the next best class.
constexpr int kGroups = 256, kList = 512;

struct TopShared {
  alignas(16) uint64_t list[kList];
  uint64_t sorted[kList];
  uint32_t group_key[kGroups], group_place[kGroups];
  uint64_t red[16];
  double wave_sum[16];
  float wave_max[16];
  int n_list;
};

// Bound of the list: the composite (value key, ~place) that at least k groups
// reach, and few more.
__device__ __forceinline__ uint64_t top_bound(const TopShared& sh, int k) {
  const int lane = threadIdx.x & 63;
  uint32_t key[4], place[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) key[i] = sh.group_key[i * 64 + lane], place[i] = sh.group_place[i * 64 + lane];
  const auto reach = [&](uint32_t t) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) n += __popcll(__ballot(key[i] >= t));
    return n;
  };
  if (reach(kNone + 1) <= k) return (uint64_t)(kNone + 1) << 32;
  uint32_t lo = max(kNone + 1, wave_min(min(min(key[0], key[1]), min(key[2], key[3]))));
  uint32_t hi = wave_max(max(max(key[0], key[1]), max(key[2], key[3]))) + 1;
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
  // Many groups tie at the bound: the first places among them.
  const int need = k - reach(lo + 1);
  uint32_t plo = 0, phi = 0xFFFFFFFFu;
  while (phi - plo > 1) {
    const uint32_t mid = plo + (phi - plo) / 2;
    int c = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) c += __popcll(__ballot(key[i] == lo && place[i] >= mid));
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

// Waves a SIMD that the registers of a part leave room for.
template <typename T, int NT, int PER, bool RULES>
constexpr int top_waves() {
  constexpr int regs = RULES ? PER * Pack<T>::N : PER * 4;
  return NT == 1024 ? 4 : regs <= 32 ? RULES ? 5 : 7 : regs <= 40 ? 6 : RULES ? 3 : 4;
}

template <typename T, int NT, int PER, bool RULES>
__global__ __launch_bounds__(NT, (top_waves<T, NT, PER, RULES>())) void top_logits_kernel(LogitRows in, TopParams p, int parts) {
  constexpr int N = Pack<T>::N, W = NT / 64;
  __shared__ TopShared sh;
  extern __shared__ int counts[];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(in.x) + row * in.stride;
  RowRules r{};
  if constexpr (RULES) r = row_rules(p.rules, row, in.classes);
  const RowShape<N> shape(in.classes, p.last_ties);
  const float c = kLog2e / p.temperature;
  for (int i = tid; i < kList; i += NT) sh.list[i] = 0;
  if (tid == 0) sh.n_list = 0;

  // Best logit of this thread and the first place that holds it.
  RowPart<T, NT, PER, !RULES> d;
  float best = -INFINITY;
  int place = 0;
  bool nan = false;
  int nan_place = 0;
  float tail = -INFINITY;
  const auto look = [&](float m, int at) {
    const bool better = m > best;
    best = better ? m : best;
    place = better ? at : place;
  };
  const auto look_tail = [&] {
    look(tail, shape.tail_place());
    if (tail != tail && !nan) nan = true, nan_place = shape.tail_place();
  };
  for (int seg = 0; seg < parts; ++seg) {
    read_part<RULES>(d, x, r, shape, seg, counts);
    if (seg == 0) {
      tail = d.tail;
      if (shape.last) look_tail();
    }
    bool bad = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      look(pack_max(d.pack[j]), shape.pack_place((seg * PER + j) * NT + tid));
#pragma unroll
      for (int e = 0; e < N; e += 2) bad |= __builtin_isunordered(d.pack[j].get(e), d.pack[j].get(e + 1));
    }
    if (bad && !nan) {
      nan = true;
      nan_place = INT32_MAX;
#pragma unroll
      for (int j = 0; j < PER; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (d.pack[j].get(e) != d.pack[j].get(e))
            nan_place = min(nan_place, shape.pack_place((seg * PER + j) * NT + tid));
    }
  }
  if (!shape.last) look_tail();
  uint64_t mine = (uint64_t)value_key(nan ? NAN : best) << 32 | (uint32_t)~(nan ? nan_place : place);
  if constexpr (NT > kGroups) {
#pragma unroll
    for (int o = 1; o < NT / kGroups; o <<= 1) mine = max(mine, (uint64_t)__shfl_xor((unsigned long long)mine, o));
  }
  if (tid % (NT / kGroups) == 0) {
    sh.group_key[tid / (NT / kGroups)] = (uint32_t)(mine >> 32);
    sh.group_place[tid / (NT / kGroups)] = (uint32_t)mine;
  }
  __syncthreads();

  // Classes above the bound go to the list, one atomic a wave: count, reserve,
  // write.  The others' sums.
  const uint64_t bound = top_bound(sh, p.k);
  const float floor_value = key_value(bound);
  d.forget();
  float wm = -INFINITY;
  double ws = 0.0;
  for (int seg = parts - 1; seg >= 0; --seg) {
    if (seg != parts - 1) read_part<RULES>(d, x, r, shape, seg, counts);
    const auto pass = [&](float v, int at) {
      const uint32_t key = value_key(v);
      return ((uint64_t)key << 32 | (uint32_t)~at) >= bound && key > kNone;
    };
    int n = 0;
    uint32_t hit = 0;  // packs with a class above the bound in some lane
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (__any(pack_max(d.pack[j]) >= floor_value || nan)) {
        const int at = shape.pack_place((seg * PER + j) * NT + tid);
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (__any(!(d.pack[j].get(e) < floor_value))) {
            n += __popcll(__ballot(pass(d.pack[j].get(e), at)));
            hit |= 1u << j;
          }
      }
    }
    const uint64_t tails = seg == 0 ? __ballot(pass(d.tail, shape.tail_place())) : 0;
    n += __popcll(tails);
    d.forget();
    if (n) {
      int slot = 0;
      if (lane == 0) slot = atomicAdd(&sh.n_list, n);
      slot = __builtin_amdgcn_readfirstlane(slot);
      const auto put = [&](uint64_t lanes, float v, int cls) {
        const int at = slot + __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0));
        const bool mine = lanes >> lane & 1;
        if (mine && at < kList) sh.list[at] = order_key(v, cls, p.last_ties);
        slot += __popcll(lanes);
        return mine;
      };
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (hit >> j & 1) {
          const int i = (seg * PER + j) * NT + tid;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float v = d.pack[j].get(e);
            if (__any(!(v < floor_value)))
              if (put(__ballot(pass(v, shape.pack_place(i))), v, shape.pack_class(i) + e)) d.pack[j].clear(e);
          }
        }
      }
      if (tails && put(tails, d.tail, shape.tail_class())) d.tail = -INFINITY;
    }
    d.forget();
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
      // Eight keys at a time (zeros behind the last).
      for (int o = 0; o < n; o += 8)
#pragma unroll
        for (int q = 0; q < 8; ++q) rank += sh.list[o + q] > key;
      sh.sorted[rank] = key;
    }
  } else {
    search_row<T, RULES>(x, r, in.classes, p, c, counts, sh, wm, ws);
    n = p.k;
    if (lane == 0) sh.wave_max[wave] = wm, sh.wave_sum[wave] = ws;
  }
  __syncthreads();
  if (wave != 0) return;

  // The best of the list, and the rest: the list's end and the waves' sums.
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
    const double top = (double)key_value((uint32_t)__builtin_amdgcn_readfirstlane((int)(key >> 32))) * inv;
    const double e = any ? exp((double)key_value(key) * inv - top) : 0.0;
    const double whole = wave_sum(e) + (m == -INFINITY ? 0.0 : exp(rest - top));
    if (lane < p.k) {
      p.pairs[(row * p.k + lane) * 2] = any ? (float)key_class(key, p.last_ties) : -1.0f;
      p.pairs[(row * p.k + lane) * 2 + 1] = any ? (float)(e / whole) : 0.0f;
    }
  }
}

template <typename T, int NT, int PER, bool RULES>
void launch_top(const LogitRows& in, const TopParams& p, hipStream_t s) {
  constexpr int kClasses = NT * PER * Pack<T>::N;
  const size_t lds = p.rules.history ? (kWindow + 8) * sizeof(int) : 0;
  hipLaunchKernelGGL((top_logits_kernel<T, NT, PER, RULES>), dim3((unsigned)in.rows), dim3(NT), lds, s, in, p,
                     (in.classes + kClasses - 1) / kClasses);
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

}  // namespace

void launch_top_logits(const LogitRows& in, const TopParams& p, hipStream_t s) {
  if (p.rules.history || p.rules.bias || p.rules.masks)
    in.dt == DT_BF16 ? launch_top_typed<bf16, true>(in, p, s) : launch_top_typed<float, true>(in, p, s);
  else
    in.dt == DT_BF16 ? launch_top_typed<bf16, false>(in, p, s) : launch_top_typed<float, false>(in, p, s);
}

}  // namespace ppocr
