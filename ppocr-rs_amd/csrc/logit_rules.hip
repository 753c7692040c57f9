// Rules on rows of class logits: penalties, biases, masks.
#include "logit_rows.h"

namespace ppocr {
namespace {

constexpr int kThreads = 256, kChunk = 4096;

// Rules of a chunk of one row: 16 elements a thread, each read and written
// once, bound by HBM.  A pack without an allowed class is not read, and in
// place one that no rule changes is neither read nor written.  Counts of the
// history's classes in the chunk are an LDS histogram, so a chunk costs one
// pass over the row's history (from L2 after the first chunk).  2560 x 6906 fp32
// under line masks and a bias: 19 us; 256 x 131072 bf16 under masks and
// histories of up to 2000 classes: 25 us, 18 of them its bytes.
template <typename T, bool HISTORY>
__global__ __launch_bounds__(kThreads) void logit_rules_kernel(LogitRows in, RuleParams p, T* out, int64_t out_stride,
                                                               int chunk) {
  constexpr int N = Pack<T>::N, PER = kChunk / (kThreads * N);
  constexpr unsigned kAll = (1u << N) - 1;
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
    bits[j] = r.mask && i < full ? mask_bits<N>(r.mask, first + i * N) : kAll;
  }
  PackBits raw[PER];
  bool write[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = tid + j * kThreads;
    write[j] = i < full;
    raw[j] = Pack<T>::none();
    if (!in_place && write[j] && bits[j]) raw[j] = load_pack(x + i * N);
  }
  if (counted) count_history(r, first, n, counts);
  if (in_place)
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = tid + j * kThreads;
      if (write[j] && bits[j] == kAll) {
        write[j] = false;
        if (counted)
#pragma unroll
          for (int e = 0; e < N; ++e) write[j] |= counts[i * N + e] > 0;
      }
      if (write[j] && bits[j]) raw[j] = load_pack(x + i * N);
    }
  float v[PER][N];
#pragma unroll
  for (int j = 0; j < PER; ++j) Pack<T>::widen(raw[j], v[j]);
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
      load_bias<N>(r.bias + first + i * N, b);
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

template <typename T, bool HISTORY>
void launch_rules(const LogitRows& in, const RuleParams& rules, void* out, int64_t out_stride, hipStream_t s) {
  // Chunks of equal length (whole packs), at most kChunk classes.
  const int n = (in.classes + kChunk - 1) / kChunk;
  const int chunk = ((in.classes + n - 1) / n + 7) / 8 * 8;
  const dim3 grid((unsigned)in.rows, (unsigned)((in.classes + chunk - 1) / chunk));
  hipLaunchKernelGGL((logit_rules_kernel<T, HISTORY>), grid, dim3(kThreads), 0, s, in, rules, static_cast<T*>(out),
                     out_stride, chunk);
}

}  // namespace

void launch_logit_rules(const LogitRows& in, const RuleParams& rules, void* out, int64_t out_stride, hipStream_t s) {
  if (in.dt == DT_BF16)
    rules.history ? launch_rules<bf16, true>(in, rules, out, out_stride, s)
                  : launch_rules<bf16, false>(in, rules, out, out_stride, s);
  else
    rules.history ? launch_rules<float, true>(in, rules, out, out_stride, s)
                  : launch_rules<float, false>(in, rules, out, out_stride, s);
}

}  // namespace ppocr
