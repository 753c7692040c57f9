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
// Of a number (no NaN), a few operations fewer.
__device__ __forceinline__ uint32_t number_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
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

// The rules of a launch: none, biases and masks, or penalties too (whose
// counting costs registers).
enum RuleParts { kNoRules, kTables, kHistory };

// The penalties on a part in registers.  The history is counted in windows of
// classes, whole rounds of packs of a part; the row's last classes have counters
// of their own behind the window's.  Short rows take small windows, which leave
// LDS for more workgroups (10000 x 6906 fp32, top 8: 102 us against 112 in one
// window), long ones large windows, for each of which the history is read again
// (2560 x 18710: 83 us against 88 in windows of 4096).
constexpr int history_window(int part_classes) {
  return part_classes <= 2048 ? part_classes : part_classes <= 8192 ? 4096 : 8192;
}

template <typename P, int N>
__device__ __forceinline__ void penalise_part(P& d, const RowRules& r, const RowShape<N>& s, int seg, int* counts) {
  constexpr int NT = P::kThreads, PER = P::kPer, kWindow = history_window(P::kClasses), kRounds = kWindow / (NT * N);
  static_assert(kRounds >= 1 && kWindow % (NT * N) == 0, "a window is whole rounds");
  if (seg == 0 && s.full * N < s.classes) {
    __syncthreads();
    count_history(r, s.full * N, s.classes - s.full * N, counts + kWindow);
    if (s.has_tail() && counts[kWindow + threadIdx.x] > 0) d.tail = penalise(r, d.tail, counts[kWindow + threadIdx.x]);
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

// Reads a part under the rules.  Packs without an allowed class are not read.
// Threads that hold many elements read the biases of several packs at once,
// where waiting for each would keep few waves idle (10240 x 18710 fp32 under a
// bias, top 5: 205 us against 239); with fewer elements the registers are worth
// more (378 x 18710 under a bias and masks 13.5 against 15.2).
template <RuleParts RULES, typename P, typename T, int N>
__device__ __forceinline__ void read_part(P& d, const T* x, const RowRules& r, const RowShape<N>& s, int seg, int* counts) {
  constexpr int NT = P::kThreads, PER = P::kPer;
  if constexpr (RULES == kNoRules) {
    load_part(d, x, s, seg);
  } else {
    unsigned bits[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = (seg * PER + j) * NT + (int)threadIdx.x;
      bits[j] = i < s.full ? (r.mask ? mask_bits<N>(r.mask, s.pack_class(i)) : (1u << N) - 1) : 0;
    }
    load_part(d, x, s, seg, bits);
    if constexpr (RULES == kHistory)
      if (r.n_history) penalise_part(d, r, s, seg, counts);
    if (r.bias) {
      constexpr int G = PER * N > 64 ? 16 / N : 1;
      // Packs that need no bias read the table's start where several go at once.
      if (s.full > 0)
#pragma unroll
        for (int j0 = 0; j0 < PER; j0 += G) {
          float b[G][N];
#pragma unroll
          for (int j = j0; j < j0 + G && j < PER; ++j)
            if (G > 1 || bits[j])
              load_bias<N>(r.bias + (bits[j] ? s.pack_class((seg * PER + j) * NT + (int)threadIdx.x) : 0), b[j - j0]);
#pragma unroll
          for (int j = j0; j < j0 + G && j < PER; ++j)
            if (bits[j])
#pragma unroll
              for (int e = 0; e < N; ++e) d.pack[j].set(e, d.pack[j].get(e) + b[j - j0][e]);
        }
      if (seg == 0 && s.has_tail()) d.tail = d.tail + r.bias[s.tail_class()];
    }
    if (r.mask) {
#pragma unroll
      for (int j = 0; j < PER; ++j) d.pack[j].keep(bits[j]);
      if (seg == 0 && s.has_tail() && !mask_bit(r.mask, s.tail_class())) d.tail = -INFINITY;
    }
  }
}

// The k best classes of a row and the log-sum-exp of the others, one row a
// workgroup, the row read once (parts of longer rows a second time).  fp32 rows
// are bound by HBM (10240 x 18710, top 8: 133 us, 5.8 TB/s), bf16 ones and long
// lists by vector work (the same in bf16, top 8: 86 us, top 64: 122 us at 1450
// operations a wave, 80% busy, where HBM would take 70).
//
// The classes form groups, each with its best (logit, first place that holds
// it).  The k-th best group bounds the k-th best class from below, and only
// about k groups hold classes above the bound: those leave the registers for a
// list of the wave in LDS, and each finds its rank by counting the better ones
// in all lists.  What is left in the registers and the end of the ranking is the
// rest.  The bound is found by bisection over the groups' order keys, every wave
// for itself.  Lists that overflow (rows whose best classes crowd in few
// threads) or a NaN (which shows in the sums) send the row to k searches for the
// next best class.
//
// Groups: of several waves 256, each of NT / 256 threads' classes, or the
// threads themselves where a mask leaves candidates to k groups or fewer (all of
// these would be listed); of a single wave its packs, or its classes where it
// holds eight a lane.
constexpr int kSorted = 512;

template <int NT>
struct TopShared {
  static constexpr int kThreadKeys = NT > 256 ? NT : 0;
  union {
    struct {
      uint32_t key[256 + kThreadKeys], place[256 + kThreadKeys];
    } group;
    uint64_t sorted[kSorted];  // written when the groups are done with
  };
  uint64_t red[16];
  double wave_sum[16];
  float wave_max[16];
  int count[16];  // of the waves' lists
  int nan;
};
// Room of a wave's list: k groups that are a wave's packs, all of whose classes
// pass, or half of it where sixteen waves' lists of as many fp32 classes fit.
template <int NT, int N>
constexpr int top_list() {
  return NT == 1024 && N == 4 ? 256 : 512;
}
// Its distance to the next wave's, so that the lists' like places lie in
// different banks.
template <int NT, int N>
constexpr int list_stride() {
  return top_list<NT, N>() + (NT > 64 ? 4 : 0);
}

// Where the history's counters lie, in entries of the lists: behind them where a
// row may have several parts, else in their place, since the counting is done
// when the lists begin.
template <int NT, int N>
constexpr int history_at() {
  return NT == 1024 ? NT / 64 * list_stride<NT, N>() : 0;
}
template <int NT, int PER, int N, RuleParts RULES>
constexpr size_t top_lds() {
  const size_t lists = NT / 64 * list_stride<NT, N>() * sizeof(uint64_t);
  const size_t counts =
      history_at<NT, N>() * sizeof(uint64_t) + (history_window(NT * PER * N) + 8) * sizeof(int);
  return RULES == kHistory && counts > lists ? counts : lists;
}

// Bound of the list: the composite (value key, ~place) that at least k of the
// wave's groups, K a lane, reach, and few more.  0: only k groups or fewer hold
// a candidate.
template <int K>
__device__ __forceinline__ uint64_t top_bound(const uint32_t (&key)[K], const uint32_t (&place)[K], int k) {
  const auto reach = [&](uint32_t t) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) n += __popcll(lanes_where(key[i] >= t));
    return n;
  };
  int n = reach(kNone + 1);
  if (n <= k) return 0;
  uint32_t least = key[0], most = key[0];
#pragma unroll
  for (int i = 1; i < K; ++i) least = min(least, key[i]), most = max(most, key[i]);
  uint32_t lo = max(kNone + 1, wave_min(least));
  uint32_t hi = wave_max(most) + 1;
  const int enough = k + k / 8 + 4;
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
    for (int i = 0; i < K; ++i) c += __popcll(lanes_where(key[i] == lo && place[i] >= mid));
    if (c >= need)
      plo = mid;
    else
      phi = mid;
  }
  return (uint64_t)lo << 32 | plo;
}

// The slow way for any row: k searches for the best class below the last one,
// then the sums of the others, the row read each time.
template <typename T, RuleParts RULES, int NT, int WINDOW>
__device__ __forceinline__ void search_row(const T* x, const RowRules& r, int classes, const TopParams& p, float c,
                                           int* counts, TopShared<NT>& sh, float& wm, double& ws) {
  const auto each = [&](auto&& f) {
    for (int first = 0; first < classes; first += WINDOW) {
      const int n = min(WINDOW, classes - first);
      bool counted = false;
      if constexpr (RULES == kHistory) {
        counted = r.n_history > 0;
        if (counted) {
          __syncthreads();
          count_history(r, first, n, counts);
        }
      }
      for (int i = threadIdx.x; i < n; i += blockDim.x) {
        float v = ld1<T>(x + first + i);
        if constexpr (RULES != kNoRules) v = apply_rules(r, v, first + i, counted ? counts[i] : 0);
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
  wm = 0 != lanes_where(some) ? m : -INFINITY;
  ws = wave_sum(sum);
}

// Waves a SIMD that the registers of a part leave room for.
template <typename T, int NT, int PER, RuleParts RULES>
constexpr int top_waves() {
  constexpr int regs = PER * Pack<T>::N;
  if (NT == 1024) return 4;
  if (regs <= 32) return RULES == kNoRules ? 7 : 5;
  return regs <= 40 ? 5 : RULES == kNoRules ? 4 : 3;
}

template <typename T, int NT, int PER, RuleParts RULES>
__global__ __launch_bounds__(NT, (top_waves<T, NT, PER, RULES>())) void top_logits_kernel(LogitRows in, TopParams p, int parts) {
  constexpr int N = Pack<T>::N, W = NT / 64, kList = top_list<NT, N>(), kStride = list_stride<NT, N>();
  __shared__ TopShared<NT> sh;
  extern __shared__ __align__(16) uint64_t lists[];  // [W][kStride]
  int* counts = reinterpret_cast<int*>(lists + history_at<NT, N>());
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(in.x) + row * in.stride;
  RowRules r{};
  if constexpr (RULES != kNoRules) r = row_rules(p.rules, row, in.classes);
  const RowShape<N> shape(in.classes, p.last_ties);
  const float c = kLog2e / p.temperature;
  if (tid == 0) sh.nan = 0;

  // Best logit of this thread and the first place that holds it.
  RowPart<T, NT, PER, false> d;
  float high[PER];  // each pack's maximum
  float best = -INFINITY;
  int place = 0;
  float tail = -INFINITY;
  const auto look = [&](float m, int at) {
    const bool better = m > best;
    best = better ? m : best;
    place = better ? at : place;
  };
  for (int seg = 0; seg < parts; ++seg) {
    read_part<RULES>(d, x, r, shape, seg, counts);
    if (seg == 0) {
      tail = d.tail;
      if (W > 1 && shape.last) look(tail, shape.tail_place());
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      high[j] = pack_max(d.pack[j]);
      if (W > 1) look(high[j], shape.pack_place((seg * PER + j) * NT + tid));
    }
  }
  uint64_t bound;
  if constexpr (W > 1) {
    if (!shape.last) look(tail, shape.tail_place());
    uint64_t mine = (uint64_t)value_key(best) << 32 | (uint32_t)~place;
    constexpr int S = NT / 256;
    if constexpr (S > 1) {
      sh.group.key[256 + tid] = (uint32_t)(mine >> 32);
      sh.group.place[256 + tid] = (uint32_t)mine;
#pragma unroll
      for (int o = 1; o < S; o <<= 1) mine = max(mine, (uint64_t)__shfl_xor((unsigned long long)mine, o));
    }
    if (tid % S == 0) {
      sh.group.key[tid / S] = (uint32_t)(mine >> 32);
      sh.group.place[tid / S] = (uint32_t)mine;
    }
    __syncthreads();
    uint32_t keys[4], places[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) keys[i] = sh.group.key[i * 64 + lane], places[i] = sh.group.place[i * 64 + lane];
    bound = top_bound(keys, places, p.k);
    if constexpr (S > 1) {
      if (!bound) {
        uint32_t all[W], at[W];
#pragma unroll
        for (int i = 0; i < W; ++i) all[i] = sh.group.key[256 + i * 64 + lane], at[i] = sh.group.place[256 + i * 64 + lane];
        bound = top_bound(all, at, p.k);
      }
    }
  } else {
    // A single wave, whose row is one part: its packs, or its classes.
    constexpr bool kClassGroups = PER * N <= 8;
    constexpr int K = (kClassGroups ? PER * N : PER) + 1;
    uint32_t keys[K], places[K];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t at = (uint32_t)~shape.pack_place(j * NT + tid);
      if constexpr (kClassGroups) {
#pragma unroll
        for (int e = 0; e < N; ++e) keys[j * N + e] = value_key(d.pack[j].get(e)), places[j * N + e] = at;
      } else {
        keys[j] = value_key(high[j]), places[j] = at;
      }
    }
    keys[K - 1] = value_key(tail), places[K - 1] = (uint32_t)~shape.tail_place();
    bound = top_bound(keys, places, p.k);
  }
  if (!bound) bound = (uint64_t)(kNone + 1) << 32;  // every candidate

  // Classes above the bound go to the wave's list; the others' sums.
  const float floor_value = key_value(bound);
  const uint32_t floor_place = (uint32_t)bound;
  uint64_t* list = lists + wave * kStride;
  float wm = -INFINITY;
  double ws = 0.0;
  int n_wave = 0;
  for (int seg = parts - 1; seg >= 0; --seg) {
    if (seg != parts - 1) {
      read_part<RULES>(d, x, r, shape, seg, counts);
#pragma unroll
      for (int j = 0; j < PER; ++j) high[j] = pack_max(d.pack[j]);
    }
    // A class passes above the bound's value, or at it in a place that the
    // bound reaches; at least -FLT_MAX in any case.
    const auto take = [&](float v, int at, int cls) {
      bool mine = v >= floor_value;
      if (!lanes_where(mine)) return false;
      if (floor_place) mine = mine && (v > floor_value || (uint32_t)~at >= floor_place);
      const uint64_t lanes = lanes_where(mine);
      const int slot = __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, n_wave));
      if (mine) list[min(slot, kList - 1)] = (uint64_t)number_key(v) << 32 | (uint32_t)(p.last_ties ? cls : ~cls);
      n_wave += __popcll(lanes);
      return mine;
    };
    bool hits = false;
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (!lanes_where(high[j] >= floor_value)) {
        m = fmaxf(m, high[j]);
        continue;
      }
      hits = true;
      const int i = (seg * PER + j) * NT + tid;
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (take(d.pack[j].get(e), shape.pack_place(i), shape.pack_class(i) + e)) d.pack[j].clear(e);
    }
    if (seg == 0 && take(d.tail, shape.tail_place(), shape.tail_class())) d.tail = -INFINITY;
    // Terms relative to a limit of the wave's maximum: classes left in a pack
    // that gave some to the list are at most the bound.  Where they are so far
    // below it that the terms' arguments would lose digits, the maximum itself is
    // looked for.
    m = fmaxf(wave_max(fmaxf(m, d.tail)), hits ? floor_value : -INFINITY);
    double sum = part_sum(d, fminf(fmaxf(m, -FLT_MAX), FLT_MAX), c);
    if (hits && sum < 0.25) {
      m = part_max(d);
      // Limited to finite numbers: +inf then counts as an infinite term and -inf
      // as none.
      sum = part_sum(d, fminf(fmaxf(m, -FLT_MAX), FLT_MAX), c);
    }
    if (sum != sum) sh.nan = 1;
    join_sums(wm, ws, fminf(m, FLT_MAX), sum, c);
  }
  if (lane == 0) sh.wave_max[wave] = wm, sh.wave_sum[wave] = ws, sh.count[wave] = n_wave;
  // Zeros behind the list, to the next step of the ranking.
  constexpr int kStep = W > 1 ? 4 : 8;
  if (lane < kStep && n_wave + lane < kList) list[n_wave + lane] = 0;
  __syncthreads();

  int n = 0, most = 0, ends[W];
#pragma unroll
  for (int w = 0; w < W; ++w) ends[w] = n += sh.count[w], most = max(most, sh.count[w]);
  if (n <= kSorted && most <= kList && !sh.nan) {
    // W lanes a class, each with one list (10240 x 6906 fp32 under masks, top 8:
    // 67 us against 78 with a lane for all lists, 1 x 18710, top 5: 6.4 against 7.5).
    constexpr int kUnroll = W > 1 ? 1 : 2;
    for (int i = tid / W; i < n; i += 64) {
      int at = i;
#pragma unroll
      for (int w = 0; w + 1 < W; ++w) at = i >= ends[w] ? (w + 1) * kStride + i - ends[w] : at;
      const uint64_t key = lists[at];
      const uint64_t* mine = lists + tid % W * kStride;
      const int end = sh.count[tid % W];
      int rank = 0;
#pragma unroll kUnroll
      for (int o = 0; o < end; o += kStep)
#pragma unroll
        for (int q = 0; q < kStep; ++q) rank += mine[o + q] > key;
#pragma unroll
      for (int o = 1; o < W; o <<= 1) rank += __shfl_xor(rank, o);
      if (tid % W == 0) sh.sorted[rank] = key;
    }
  } else {
    search_row<T, RULES, NT, history_window(NT * PER * N)>(x, r, in.classes, p, c, counts, sh, wm, ws);
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

template <typename T, int NT, int PER, RuleParts RULES>
void launch_top(const LogitRows& in, const TopParams& p, hipStream_t s) {
  constexpr int kClasses = NT * PER * Pack<T>::N;
  constexpr size_t lds = top_lds<NT, PER, Pack<T>::N, RULES>();
  hipLaunchKernelGGL((top_logits_kernel<T, NT, PER, RULES>), dim3((unsigned)in.rows), dim3(NT), lds, s, in, p,
                     (in.classes + kClasses - 1) / kClasses);
}

// Threads of a row's workgroup and the elements that each holds.  Short rows
// take a wave, which waits for no other (20000 x 300 fp32, top 64: 49 us against
// 111 with 256 threads), with 32 elements a thread where there are rows enough
// to hide its latency (10000 x 1900, top 8: 31 us against 48; 300 x 1000 10
// against 8.7).  A few hundred rows fill the chip better with 512 threads (378 x
// 18710 fp32 under masks, top 3: 14.5 us against 20.4 with 1024), batches with
// 256, where fewer waves repeat the search for the bound (10240 x 18710 fp32,
// top 64: 149 us against 223 with 512).  Longer rows are read twice in parts
// rather than held by 1024 threads, whose one workgroup leaves its CU idle at
// each wait (700 x 70000 fp32: 52 us against 57, 1500 x 30001 in one part 42
// against 80 then, 37 now), but where rules would be applied twice too (256 x 131072 under
// masks 37 against 54) or few rows leave CUs idle.
template <typename T, RuleParts RULES>
void launch_top_rules(const LogitRows& in, const TopParams& p, hipStream_t s) {
  constexpr int N = Pack<T>::N, kLong = RULES != kNoRules ? 64 : 80;
  if (in.classes <= 64 * 8)
    launch_top<T, 64, 8 / N, RULES>(in, p, s);
  else if (in.rows >= 1024 && in.classes <= 64 * 32)
    launch_top<T, 64, 32 / N, RULES>(in, p, s);
  else if (in.rows < 1024 && in.classes > 64 * 32 && in.classes <= 512 * 40)
    launch_top<T, 512, 40 / N, RULES>(in, p, s);
  else if (in.classes <= 256 * 32)
    launch_top<T, 256, 32 / N, RULES>(in, p, s);
  else if (in.classes <= 256 * 80)
    launch_top<T, 256, 80 / N, RULES>(in, p, s);
  else if (in.classes <= 512 * 80 || (RULES == kNoRules && in.rows >= 256))
    launch_top<T, 512, 80 / N, RULES>(in, p, s);
  else
    launch_top<T, 1024, kLong / N, RULES>(in, p, s);
}

template <typename T>
void launch_top_typed(const LogitRows& in, const TopParams& p, hipStream_t s) {
  if (p.rules.history)
    launch_top_rules<T, kHistory>(in, p, s);
  else if (p.rules.bias || p.rules.masks)
    launch_top_rules<T, kTables>(in, p, s);
  else
    launch_top_rules<T, kNoRules>(in, p, s);
}

}  // namespace

void launch_top_logits(const LogitRows& in, const TopParams& p, hipStream_t s) {
  in.dt == DT_BF16 ? launch_top_typed<bf16>(in, p, s) : launch_top_typed<float>(in, p, s);
}

}  // namespace ppocr
