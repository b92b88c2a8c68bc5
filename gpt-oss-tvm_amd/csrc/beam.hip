// Beam search's selection (gfx950): the k best of a request's beams x vocabulary continuations.
//
// The score of (beam b, token t) is scores[b] + x_t - log sum exp(x), x the beam's logits, in
// fp64; a beam whose logits have no maximum (NaN, +inf, nothing but -inf), or a score that is NaN,
// gives -inf.  The order is by score, then beam, then token, ascending.
#include <type_traits>

#include "moe_common.h"

namespace beam {

using moe::bf2f;

constexpr int kThreads = 1024;

template <class T>
__device__ __forceinline__ float logit(const T* x, int i) {
  if constexpr (sizeof(T) == 2) return bf2f(x[i]);
  return x[i];
}

// maximum and log of the sum of exp(x - maximum) of each row
template <class T>
__global__ __launch_bounds__(kThreads) void stats_kernel(const T* __restrict__ logits, int V,
                                                         double* __restrict__ stats) {
  __shared__ double tmp[kThreads / 64];
  const T* x = logits + (size_t)blockIdx.x * V;
  const int t = threadIdx.x;
  float m = -INFINITY;
  for (int i = t; i < V; i += kThreads) {
    const float v = logit(x, i);
    m = v != v ? INFINITY : fmaxf(m, v);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
  if ((t & 63) == 0) tmp[t >> 6] = m;
  __syncthreads();
  for (int i = 0; i < kThreads / 64; ++i) m = fmaxf(m, (float)tmp[i]);
  __syncthreads();
  double s = 0.0;
  for (int i = t; i < V; i += kThreads) s += exp((double)logit(x, i) - (double)m);
  s = moe::wave_sum(s);
  if ((t & 63) == 0) tmp[t >> 6] = s;
  __syncthreads();
  if (t == 0) {
    s = 0.0;
    for (int i = 0; i < kThreads / 64; ++i) s += tmp[i];
    stats[2 * blockIdx.x] = m;
    stats[2 * blockIdx.x + 1] = log(s);
  }
}

// the k best of a request, one after the other: each the best of those behind the last
template <class T>
__global__ __launch_bounds__(kThreads) void select_kernel(
    const T* __restrict__ logits, const float* __restrict__ scores, int W, int V, int k,
    const double* __restrict__ stats, float* __restrict__ out_scores, int* __restrict__ out_beams,
    int* __restrict__ out_tokens) {
  __shared__ double bv[kThreads / 64];
  __shared__ int64_t bi[kThreads / 64];
  const int r = blockIdx.x, t = threadIdx.x;
  double last_v = INFINITY;
  int64_t last_i = -1;
  auto before = [](double v, int64_t i, double w, int64_t j) { return v > w || (v == w && i < j); };
  for (int n = 0; n < k; ++n) {
    double best = -INFINITY;
    int64_t at = INT64_MAX;
    for (int b = 0; b < W; ++b) {
      const double m = stats[2 * (r * W + b)], lse = stats[2 * (r * W + b) + 1];
      const double score = scores[r * W + b];
      const T* x = logits + (size_t)(r * W + b) * V;
      for (int i = t; i < V; i += kThreads) {
        double v = score + (((double)logit(x, i) - m) - lse);
        if (v != v) v = -INFINITY;
        const int64_t idx = (int64_t)b * V + i;
        if (before(last_v, last_i, v, idx) && before(v, idx, best, at)) {
          best = v;
          at = idx;
        }
      }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      const double v = __shfl_xor(best, off, 64);
      const int64_t i = __shfl_xor(at, off, 64);
      if (before(v, i, best, at)) {
        best = v;
        at = i;
      }
    }
    if ((t & 63) == 0) {
      bv[t >> 6] = best;
      bi[t >> 6] = at;
    }
    __syncthreads();
    for (int i = 0; i < kThreads / 64; ++i)
      if (before(bv[i], bi[i], best, at)) {
        best = bv[i];
        at = bi[i];
      }
    __syncthreads();
    last_v = best;
    last_i = at;
    if (t == 0) {
      out_scores[r * k + n] = (float)best;
      out_beams[r * k + n] = (int)(at / V);
      out_tokens[r * k + n] = (int)(at % V);
    }
  }
}

}  // namespace beam

extern "C" {

size_t attn_beam_state_bytes(int rows, int vocab, int k) { return (size_t)rows * 16; }

int attn_launch_beam(const void* logits, bool f32, const float* scores, int batch, int width,
                     int vocab, int k, float* out_scores, int* out_beams, int* out_tokens,
                     void* state, hipStream_t s) {
  double* stats = (double*)state;
  auto go = [&](auto* x) {
    using T = std::remove_pointer_t<decltype(x)>;
    hipLaunchKernelGGL((beam::stats_kernel<std::remove_const_t<T>>), dim3(batch * width),
                       dim3(beam::kThreads), 0, s, x, vocab, stats);
    if (hipGetLastError() != hipSuccess) return -6;
    hipLaunchKernelGGL((beam::select_kernel<std::remove_const_t<T>>), dim3(batch),
                       dim3(beam::kThreads), 0, s, x, scores, width, vocab, k, stats, out_scores,
                       out_beams, out_tokens);
    return hipGetLastError() == hipSuccess ? 0 : -6;
  };
  return f32 ? go((const float*)logits) : go((const uint16_t*)logits);
}

}  // extern "C"
