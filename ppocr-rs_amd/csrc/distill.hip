// Distillation of rows of class logits from a teacher's best classes.
#include "logit_rows.h"

namespace ppocr {
namespace {

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

// Distillation of one row a workgroup: its loss, its gradient, or both.
//
// With e_c = exp((s_c - M) / tau), Z0 the sum of e over the classes that are no
// entry, Z = Z0 + sum over the entries, p = e / Z and the rest's share of the
// student p0 = Z0 / Z:
//   loss = tau^2 (sum_j q_j (log q_j - log p_j) + q0 (log q0 - log p0)),
//   d loss / d s_c = tau (p_c - q_c) for an entry, tau e_c (1 / Z - q0 / Z0) else.
// So the rest's gradient is e times one factor of the row, and the row is read
// once: it stays in registers with the entries taken out (by marks in LDS).
// Wave 0 does the entries, in 64 bits (the loss is a difference of logs that
// nearly cancel), the teacher's shares while the row is on its way, and writes
// their gradients over the row's; scalars of the row take lanes of the same
// exponentials and logarithms, of which a batch of short rows would else do
// little more.  The whole is formed from the rest and the entries, so that the
// shares add up to one and an error of the rest's sum cancels to first order in
// the loss.  Rows longer than the registers go through them in parts, twice when
// the gradient is asked for.
enum DistillMode { kLoss, kBoth, kGradient };

struct DistillShared {
  double sum[16];
  float max[16];
  float factor, top;  // of the rest's gradient: exp((s - top) / tau) times factor
  // The teacher's shares q, which wave 0 keeps here rather than in registers:
  // log q = level - log(whole).
  double q[64], level[64];
  double q0, level0, whole;
};

// Whether bf16 rows stay as stored in the registers, widened anew by each pass:
// where the row lives through both passes the waves that this leaves room for
// are worth more than the operations (10240 x 18710, loss and gradient: 158 us
// against 177; 256 x 131072 in parts 38 against 35; the loss alone of 10240 x
// 6906 45 against 41).
template <typename T, int PER, bool PARTS, DistillMode MODE>
constexpr bool distill_raw() {
  return PER * Pack<T>::N > 40 || (MODE == kBoth && !PARTS);
}

// Waves a SIMD that the registers of a part leave room for.
template <int PER>
constexpr int distill_waves() {
  return PER * 4 <= 16 ? 8 : 5;
}

__device__ __forceinline__ double lane_value(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// The teacher's shares of a row, by wave 0.  An entry that does not count loses
// its index.
__device__ __forceinline__ void teacher_shares(const DistillParams& p, int64_t row, TeacherEntry& entry, double inv,
                                               bool maybe_again, DistillShared& sh) {
  const int lane = threadIdx.x & 63;
  // A class named twice counts once, with its first entry.
  bool again = false;
  for (int j = 0; maybe_again && j + 1 < p.k; ++j)
    again |= __builtin_amdgcn_readlane(entry.index, j) == entry.index && j < lane;
  if (again) entry.index = -1;
  const bool valid = entry.index >= 0;
  const double rest = p.rest ? (double)p.rest[row] : -INFINITY;
  const double m = fmax((double)wave_max(valid ? entry.value : -INFINITY) * inv, rest);
  const double d = (double)entry.value * inv - m, d0 = rest - m;
  // The rest takes the last lane where it holds no entry.
  const bool spare = p.k < 64;
  const double x = exp(spare && lane == 63 ? d0 : d);
  const double x0 = spare ? lane_value(x, 63) : exp(d0);
  const double whole = wave_sum(valid ? x : 0.0) + x0, share = 1.0 / whole;
  sh.q[lane] = valid ? x * share : 0.0;
  sh.level[lane] = d;
  if (lane == 0) sh.q0 = x0 * share, sh.level0 = d0, sh.whole = whole;
}

// Marks of the entries' classes below the row's last classes % N: a bit a class,
// for all parts of a row at once, so that the waves run through the parts
// without waiting for each other (256 x 131072 fp32, loss: 29.4 us against 44
// with marks by the part).  An fp32 row of one part has a byte a pack instead, a
// thread's bytes together, so that a thread reads four packs' marks at once
// (10240 x 18710, loss: 126 us against 144); in bf16, with half as many packs,
// bits are faster (92 us against 98).
template <int N, int NT, int PER, bool PARTS>
struct Marks {
  static constexpr bool kBits = PARTS || N == 8;
  static constexpr int kWords = (PER + 3) / 4;
  const RowShape<N>& shape;
  uint32_t* at;

  static size_t words(int classes) { return kBits ? (size_t)(classes + 31) / 32 : (size_t)NT * kWords; }
  __device__ __forceinline__ void reset() {
    if constexpr (kBits) {
      for (int i = threadIdx.x; i < (shape.classes + 31) / 32; i += NT) at[i] = 0;
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) at[threadIdx.x * kWords + i] = 0;
    }
  }
  // Marks a class; whether it may have been marked before.
  __device__ __forceinline__ bool set(int c) {
    const int i = c / N;
    if (i >= shape.full) return true;
    const int word = kBits ? c >> 5 : i % NT * kWords + (i / NT >> 2);
    const uint32_t bit = 1u << (kBits ? c & 31 : (i / NT & 3) * 8 + c % N);
    return (atomicOr(&at[word], bit) & bit) != 0;
  }
  // Takes the marked classes out of a part.
  template <typename P>
  __device__ __forceinline__ void clear(P& d, int seg) const {
    if constexpr (kBits) {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = (seg * PER + j) * NT + (int)threadIdx.x;
        const unsigned bits = i < shape.full ? mask_bits<N>(at, i * N) : 0;
        if (bits) d.pack[j].drop(bits);
      }
    } else {
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        const uint32_t word = at[threadIdx.x * kWords + w];
        if (word)
#pragma unroll
          for (int q = 0; q < 4 && w * 4 + q < PER; ++q) d.pack[w * 4 + q].drop(word >> (q * 8));
      }
    }
  }
};

// PARTS: rows of `parts` parts; else the whole row is one.
template <typename T, int NT, int PER, bool PARTS, DistillMode MODE>
__global__ __launch_bounds__(NT, distill_waves<PER>()) void distill_kernel(LogitRows s, DistillParams p, int parts) {
  constexpr int N = Pack<T>::N, W = NT / 64;
  __shared__ DistillShared sh;
  extern __shared__ uint32_t mark_words[];  // not of the gradient alone
  const int segs = PARTS ? parts : 1;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const RowShape<N> shape(s.classes, 0);
  const T* x = static_cast<const T*>(s.x) + row * s.stride;
  T* g = static_cast<T*>(p.grad) + row * p.grad_stride;
  TeacherEntry entry = teacher_entry(p, row, s.classes);
  if (!lanes_where(entry.index >= 0)) {
    if (MODE != kGradient && tid == 0) p.loss[row] = 0.0f;
    if (MODE == kLoss && p.state && tid < 4) p.state[row * 4 + tid] = 0.0f;
    if (MODE != kLoss) {
      const float zero[N] = {};
      for (int i = tid; i < shape.full; i += NT) Pack<T>::store(g + i * N, zero);
      if (shape.has_tail()) st1<T>(g + shape.tail_class(), 0.0f);
    }
    return;
  }
  const float c = kLog2e / p.temperature;
  const double inv = 1.0 / (double)p.temperature;
  // The entries' own logits, before a gradient in place covers them.
  float own = 0.0f;
  if (wave == 0 && entry.index >= 0) own = ld1<T>(x + entry.index);

  RowPart<T, NT, PER, distill_raw<T, PER, PARTS, MODE>()> d;
  float m = -INFINITY;  // the wave's maximum and sum of the rest
  double sum = 0.0;
  if (!PARTS || MODE != kGradient) load_part(d, x, shape, 0);
  if constexpr (MODE != kGradient) {
    Marks<N, NT, PER, PARTS> marks{shape, mark_words};
    marks.reset();
    __syncthreads();
    bool again = false;  // whether a class may be named twice
    if (wave == 0 && entry.index >= 0) again = marks.set(entry.index);
    __syncthreads();
    if (wave == 0) teacher_shares(p, row, entry, inv, lanes_where(again) != 0, sh);
    for (int seg = 0; seg < segs; ++seg) {
      if (seg > 0) load_part(d, x, shape, seg);
      marks.clear(d, seg);
      if (seg == 0 && lanes_where(entry.index >= shape.full * N)) {
        // Entries among the row's last classes, one a thread.
        for (int j = 0; j < p.k; ++j)
          if (__builtin_amdgcn_readlane(entry.index, j) == shape.tail_class()) d.tail = -INFINITY;
      }
      float pm = part_max(d);
      const double ps = part_sum(d, fmaxf(pm, -FLT_MAX), c);
      if (ps != ps) pm = fmaxf(pm, -FLT_MAX);  // a NaN is no maximum but must not be lost
      if (PARTS)
        join_sums(m, sum, pm, ps, c);
      else
        m = pm, sum = ps;
    }
    if (lane == 0) sh.max[wave] = m, sh.sum[wave] = sum;
    __syncthreads();
  }

  float entry_grad = 0.0f;
  if (wave == 0) {
    if constexpr (MODE == kGradient) teacher_shares(p, row, entry, inv, true, sh);
    const bool valid = entry.index >= 0;
    const double q = sh.q[lane], q0 = sh.q0;
    double top, z, mr, zr;
    float om = -INFINITY;
    if constexpr (MODE == kGradient) {
      const float* st = p.state + row * 4;
      top = st[0], z = st[1], mr = st[2], zr = st[3];
    } else {
      if (lane < W) om = sh.max[lane];
      mr = wave_max(om);
      top = fmaxf((float)mr, wave_max(valid ? own : -INFINITY));
    }
    const double low = fmax(top, -(double)FLT_MAX);
    const double a = ((double)own - low) * inv, a0 = (mr - low) * inv;
    const double e = valid ? exp(a) : 0.0;
    // Of the rest's maximum in the last lane, of the waves' in theirs.
    const double joint = exp(lane < W ? ((double)om - mr) * inv : a0);
    const double e0 = mr == -INFINITY ? 0.0 : lane_value(joint, 63);
    if constexpr (MODE != kGradient) {
      zr = wave_sum(om > -INFINITY ? sh.sum[lane] * joint : 0.0);
      z = wave_sum(e) + zr * e0;
      const double logs = log(lane == 0 ? z : lane == 1 ? zr : sh.whole);
      const double logz = lane_value(logs, 0), logzr = lane_value(logs, 1), logwhole = lane_value(logs, 2);
      double term = valid && q > 0.0 ? q * (sh.level[lane] - logwhole - (a - logz)) : 0.0;
      if (lane == 0 && q0 > 0.0)
        term += q0 * (sh.level0 - logwhole - (zr > 0.0 || zr != zr ? a0 + logzr - logz : -INFINITY));
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
      const double share = 1.0 / z;
      const double factor = dead || zr == 0.0 ? 0.0 : scale * (e0 * share - q0 / zr);
      entry_grad = dead ? 0.0f : (float)(scale * (e * share - q));
      if (lane == 0) sh.factor = (float)factor, sh.top = (float)fmax(mr, -(double)FLT_MAX);
    }
  }
  if constexpr (MODE != kLoss) {
    __syncthreads();
    const float factor = sh.factor, ref = sh.top;
    d.forget();
    for (int seg = segs - 1; seg >= 0; --seg) {
      if (PARTS) load_part(d, x, shape, seg);
      // By the difference: this loop's two forms would share their addresses,
      // which then take the registers.
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = (seg * PER + j) * NT + tid;
        if (i >= shape.full) continue;
        float v[N];
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = factor * __builtin_amdgcn_exp2f((d.pack[j].get(e) - ref) * c);
        Pack<T>::store(g + i * N, v);
      }
      if (seg == 0 && shape.has_tail())
        st1<T>(g + shape.tail_class(), factor * __builtin_amdgcn_exp2f((d.tail - ref) * c));
    }
    __syncthreads();
    if (wave == 0 && entry.index >= 0) st1<T>(g + entry.index, entry_grad);
  }
}

template <typename T, int NT, int PER, bool PARTS, DistillMode MODE>
void launch_distill_one(const LogitRows& in, const DistillParams& p, hipStream_t s) {
  constexpr int kClasses = NT * PER * Pack<T>::N;
  const size_t lds = MODE == kGradient ? 0 : Marks<Pack<T>::N, NT, PER, PARTS>::words(in.classes) * sizeof(uint32_t);
  hipLaunchKernelGGL((distill_kernel<T, NT, PER, PARTS, MODE>), dim3((unsigned)in.rows), dim3(NT), lds, s, in, p,
                     (in.classes + kClasses - 1) / kClasses);
}

// Threads of a row's workgroup and the elements that each holds.  Short rows
// take a wave, which waits for no other (20000 x 300 fp32, loss: 26 us against
// 59 with 256 threads, 10000 x 1900 20 against 34; 40 x 1900 bf16 7.4 against
// 7.0).  Else 512 threads
// of 40 elements keep more waves on a CU than 256 of 80 (2560 x 18710 fp32, loss
// and gradient: 80 us against 105), but for the loss alone of bf16 batches,
// whose rows take half the registers (10240 x 18710: 92 us against 109).  Now
// 2560 x 18710 fp32: loss 31.5 us (6.1 TB/s), gradient 75 us (5.1), both 79 us
// (4.9); 10240 x 18710 bf16: 81 us (4.8), 140 us (5.5), 157 us (4.9).
template <typename T, DistillMode MODE>
void launch_distill_typed(const LogitRows& in, const DistillParams& p, hipStream_t s) {
  constexpr int N = Pack<T>::N;
  if constexpr (MODE == kLoss && sizeof(T) == 2)
    if (in.rows >= 1024 && in.classes > 256 * 32 && in.classes <= 256 * 80)
      return launch_distill_one<T, 256, 80 / N, false, MODE>(in, p, s);
  if (in.classes <= 64 * 8)
    launch_distill_one<T, 64, 8 / N, false, MODE>(in, p, s);
  else if (in.classes <= 64 * 32)
    launch_distill_one<T, 64, 32 / N, false, MODE>(in, p, s);
  else if (in.classes <= 256 * 8 || (in.rows >= 1024 && in.classes <= 256 * 32))
    launch_distill_one<T, 256, 32 / N, false, MODE>(in, p, s);
  else if (in.classes <= 512 * 40)
    launch_distill_one<T, 512, 40 / N, false, MODE>(in, p, s);
  else if (in.classes <= 1024 * 40)
    launch_distill_one<T, 1024, 40 / N, false, MODE>(in, p, s);
  else
    launch_distill_one<T, 1024, 40 / N, true, MODE>(in, p, s);
}

template <DistillMode MODE>
void launch_distill_mode(const LogitRows& in, const DistillParams& p, hipStream_t s) {
  in.dt == DT_BF16 ? launch_distill_typed<bf16, MODE>(in, p, s) : launch_distill_typed<float, MODE>(in, p, s);
}

}  // namespace

void launch_distill(const LogitRows& student, const DistillParams& p, hipStream_t s) {
  p.grad ? launch_distill_mode<kBoth>(student, p, s) : launch_distill_mode<kLoss>(student, p, s);
}

void launch_distill_grad(const LogitRows& student, const DistillParams& p, hipStream_t s) {
  launch_distill_mode<kGradient>(student, p, s);
}

}  // namespace ppocr
