// Beam search's selection (gfx950): the k best of a request's beams x vocabulary continuations.
//
// The score of (beam b, token t) is scores[b] + x_t - log sum exp(x), x the beam's logits, in
// fp64 but for the exponentials (fp32, added up sixteen at a time); a beam whose logits have no
// maximum (NaN, +inf, nothing but -inf), or whose own score is not finite, gives -inf.  The order
// is by score, then beam, then logit, then token.
//
// Two launches.  part_kernel reads the logits once, a workgroup a stretch of a row: its maximum m,
// the sum of exp(x - m), and its k best by logit (within a row the order is the logits').
// merge_kernel, a workgroup a request, joins the sums and picks the k best of all stretches' lists.
// Both find a bound first.  Of q waves that hold numbers, each takes the ceil(k / q)-th largest
// of its lanes' maxima, by bits from above with a ballot each: where q waves reach a bound there
// are k numbers that do.  With q half of the waves (and the q-th largest of their values) about 2 k
// numbers of a stretch reach it, with q = 1 ten times k.  They go to LDS, and take their
// places by counting those before them.
//
// What bounds it, us of the two launches at rows of 201088: 128 bf16 rows (51 MB, k = 16) 16.7 +
// 6.0, 20 fp32 rows (16 MB, k = 10) 9 + 6.4, 4 bf16 rows (k = 8) 6.5 + 5.5.  The first is 3.1 TB/s:
// a pass that only reads takes 10.6, the exponentials, bounds and lists the rest.  Few rows: loads
// and barriers that wait for one another, in both launches.
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "moe_common.h"

namespace beam {

using moe::u32x4;
using moe::u32x4_any;

constexpr int kMost = 64;        // k at most: the lanes of a wave
constexpr int kBoundBits = 18;   // of the bounds: 2^-9 of a value lets few more through

struct Stat {  // of a stretch
  double sum;  // of exp(x - m), m = 0 where there is nothing but -inf
  float m;
};
struct Item {
  float x;
  int token;  // -1: none
};

// order-preserving image of a float (both zeros alike)
__device__ __forceinline__ uint32_t image(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// a bound on the k-th largest of a wave's values from below: its upper kBits bits
template <int kBits, class U>
__device__ __forceinline__ U kth_of_lanes(U mine, int k) {
  constexpr int kAll = 8 * sizeof(U);
  U t = 0u;
#pragma unroll
  for (int bit = kAll - 1; bit >= kAll - kBits; --bit) {
    const U next = t | (U)1 << bit;
    if (__popcll(__ballot(mine >= next)) >= k) t = next;
  }
  return t;
}
// the q-th largest of n values, n <= 64, q <= n
__device__ __forceinline__ uint32_t nth_of(const uint32_t* x, int n, int q) {
  const int lane = threadIdx.x & 63;
  const uint32_t mine = x[min(lane, n - 1)];
  int before = 0;
  for (int i = 0; i < n; ++i) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)mine, i);
    before += o > mine || (o == mine && i < lane) ? 1 : 0;
  }
  return (uint32_t)__builtin_amdgcn_readlane(
      (int)mine, __builtin_ctzll(__ballot(lane < n && before == q - 1)));
}
// max over the wave, by register moves: pairs, quads, rows of 16, then across the rows
template <int kCtrl, int kRows>
__device__ __forceinline__ float max_with(float x) {
  const int u = __float_as_int(x);
  return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(u, u, kCtrl, kRows, 0xF, false)));
}
__device__ __forceinline__ float wave_max(float x) {
  x = max_with<0xB1, 0xF>(x);   // quad_perm [1,0,3,2]
  x = max_with<0x4E, 0xF>(x);   // quad_perm [2,3,0,1]
  x = max_with<0x141, 0xF>(x);  // row_half_mirror
  x = max_with<0x140, 0xF>(x);  // row_mirror
  x = max_with<0x142, 0xA>(x);  // row_bcast:15 into rows 1 and 3
  x = max_with<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// Adds to ranks[i] how many of n things come before thing i: the fewer things, the more threads
// share out one's comparisons.
template <int kThreads, class At, class Before>
__device__ __forceinline__ void rank_all(int n, int* ranks, At at, Before before) {
  const int t = threadIdx.x;
  int share = 1;  // threads a thing
  while (share < 16 && n * share * 2 <= kThreads) share *= 2;
  const int step = kThreads / share, from = t / step;
  for (int i = t % step; i < n; i += step) {
    const auto mine = at(i);
    int rank = 0;
    for (int j = from; j < n; j += share) rank += before(at(j), mine) ? 1 : 0;
    if (rank) atomicAdd(&ranks[i], rank);
  }
}

// exp(d): off by up to (2 + 1.3 |d|) 2^-24 of itself (the instruction's step, the product's half of
// one, log2(e)'s own rounding)
__device__ __forceinline__ float exp_of(float d) {
  return __builtin_amdgcn_exp2f(d * 1.44269502f);
}

// T: float or uint16_t (bf16).  A stretch is `chunks` chunks, of which a thread holds 16 elements
// and the next one's loads, wherever the row begins.  The bound is taken after the first, then
// after 8, 16, .. and after the last; a thread whose maximum of a chunk reaches it only notes that
// (looking at each number there cost twice the time), and what reaches the last bound is picked out
// of the noted ones' 16 numbers, from memory, at the end.
constexpr int kPartThreads = 512, kPartElems = 16, kChunk = kPartThreads * kPartElems;
constexpr int kPartList = 1024, kWaveList = kPartList / (kPartThreads / 64);
template <class T>
__global__ __launch_bounds__(kPartThreads) __attribute__((amdgpu_waves_per_eu(6))) void part_kernel(
    const T* __restrict__ logits, int V, int k, int parts, int chunks, Stat* __restrict__ stats,
    Item* __restrict__ items) {
  constexpr int kEach = 16 / sizeof(T), kElems = kPartElems, kLoads = kElems / kEach;
  constexpr int kWaves = kPartThreads / 64;
  __shared__ int found[kWaves][kWaveList];  // (chunk, thread) whose maximum reached the bound
  __shared__ Item list[kPartList];
  __shared__ int ranks[kPartList], kept;
  __shared__ double wsum[kWaves];
  __shared__ float wm[kWaves];
  __shared__ uint32_t wbound[2][kWaves];
  __shared__ int wcount[2][kWaves];
  const int part = blockIdx.x % parts, t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const T* const x = logits + (size_t)(blockIdx.x / parts) * V;
  const int begin = part * chunks * kChunk, end = min(V, begin + chunks * kChunk);
  struct Raw {
    u32x4 w[kLoads];
    __device__ __forceinline__ float operator()(int e) const {
      const uint32_t u = w[e / kEach][sizeof(T) == 2 ? (e % kEach) >> 1 : e % kEach];
      if constexpr (sizeof(T) == 2) return __uint_as_float(e & 1 ? u & 0xFFFF0000u : u << 16);
      return __uint_as_float(u);
    }
  };
  // The stretch's whole 16-byte units are loaded without a branch (one would wait for its load
  // before the next), past the last the last again, which then counts as -inf; the few numbers
  // behind them have a thread each.
  const int units = (end - begin) / kEach, tail = end - begin - units * kEach;
  auto load = [&](Raw& raw, int chunk) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int u = min((chunk * kLoads + j) * kPartThreads + t, units - 1);
      raw.w[j] = *(const u32x4_any*)(x + begin + u * kEach);
    }
  };
  auto outside = [&](Raw& raw, int chunk) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const bool in = (chunk * kLoads + j) * kPartThreads + t < units;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        raw.w[j][w] = in ? raw.w[j][w] : sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;
    }
  };
  auto number = [&](int p) {
    return sizeof(T) == 2 ? moe::bf2f((uint16_t)x[p]) : (float)x[p];
  };
  Raw raw, next;
  if (units > 0) load(raw, 0);
  const float extra = t < tail ? number(end - tail + t) : -INFINITY;
  for (int i = t; i < kPartList; i += kPartThreads) ranks[i] = 0;
  // The lane's maximum (it passes over NaN; the sum does not) and sum of exp(x - base).  Each
  // chunk's sixteen are added up in fp32 by fours and go to an fp64 sum: in an fp32 one of a whole row
  // (201088 numbers, few distinct) the logarithm was off by 2e-5.  The base is a maximum of the
  // lane's and is renewed where a chunk's is more than 1 above: as many rescalings then lie
  // behind a number as its exponent is low, however the row ascends.
  float lm = fmaxf(extra, -INFINITY), base = lm, least = -INFINITY;
  double s = exp_of(extra - (lm == -INFINITY ? 0.0f : lm));
  int noted = 0;  // by the wave
  // waves with fewer numbers than lanes are not counted on for the bound
  const int full = min(kWaves, max(1, (end - begin) / (64 * kEach))), q = (full + 1) / 2;
  auto bound = [&](auto bits, int turn) __attribute__((always_inline)) {
    const uint32_t mine = kth_of_lanes<decltype(bits)::value>(image(lm), (k + q - 1) / q);
    if (lane == 0) wbound[turn][wave] = mine;
    __syncthreads();
    const uint32_t top = nth_of(wbound[turn], kWaves, q);
    // the image back, where there are k numbers (below -inf's image it would be a NaN)
    least = top <= 0x007FFFFFu
                ? -INFINITY : __uint_as_float(top & 0x80000000u ? top & 0x7FFFFFFFu : ~top);
  };
  constexpr std::integral_constant<int, kBoundBits> coarse;
  int chunk = 0;
  for (; chunk * kLoads * kPartThreads < units; ++chunk) {
    load(next, chunk + 1);
    if ((chunk + 1) * kLoads * kPartThreads > units) outside(raw, chunk);
    float cm = -INFINITY;
#pragma unroll
    for (int e = 0; e < kElems; ++e) cm = fmaxf(cm, raw(e));
    const float old = base;
    base = cm > old + 1.0f ? cm : old;
    lm = fmaxf(lm, cm);
    const float from = base == -INFINITY ? 0.0f : base;
    float four[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < kElems; ++e) four[e & 3] += exp_of(raw(e) - from);
    s = s * (double)exp_of(old - from) + (double)((four[0] + four[1]) + (four[2] + four[3]));
    if ((chunk & (chunk + 1)) == 0 && (chunk == 0 || chunk >= 7))
      bound(coarse, __builtin_ctz(chunk + 1) & 1);
    const uint64_t who = __ballot(cm >= least);
    const int at = noted + __builtin_amdgcn_mbcnt_hi(
                               (uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0u));
    if (cm >= least && at < kWaveList) found[wave][at] = chunk * kPartThreads + t;
    noted += __popcll(who);
    raw = next;
  }
  if (t == 0) kept = 0;
  float m = wave_max(lm);
  if (lane == 0) {
    wm[wave] = m;
    wcount[0][wave] = noted;
  }
  if (chunk == 1 && tail == 0)
    __syncthreads();  // (as it was taken)
  else
    bound(coarse, chunk < 8 ? 1 : (32 - __builtin_clz(chunk)) & 1);  // (not the last one's turn)
  bool fits = true;
  int records = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    m = fmaxf(m, wm[w]);
    records += wcount[0][w];
    fits = fits && wcount[0][w] <= kWaveList;
  }
  auto keep = [&](float v, int p) {  // (in any order: their places are found by comparing)
    const int at = atomicAdd(&kept, 1);
    if (at < kPartList) list[at] = Item{v, p};
  };
  if (fits) {
    for (int i = t; i < records * kLoads; i += kPartThreads) {
      int r = i / kLoads, w = 0;
      for (; r >= wcount[0][w]; ++w) r -= wcount[0][w];
      const int note = found[w][r];
      const int u =
          (note / kPartThreads * kLoads + i % kLoads) * kPartThreads + note % kPartThreads;
      if (u >= units) continue;
      Raw again;
      again.w[0] = *(const u32x4_any*)(x + begin + u * kEach);
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (again(e) >= least) keep(again(e), begin + u * kEach + e);
    }
    if (t < tail && extra >= least) keep(extra, end - tail + t);
  }
  const double sum = moe::wave_sum_f64(base == -INFINITY ? s : s * (double)exp_of(base - m));
  if (lane == 0) wsum[wave] = sum;
  __syncthreads();
  if (t == 0) {
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all += wsum[w];
    stats[blockIdx.x] = Stat{all, m};
  }
  int n = kept;
  bool chosen = fits && n <= kPartList;
  if (!chosen) {
    // Too many reach a bound (most logits equal, as where a mask leaves few tokens, or a row in
    // ascending order): with the last bound exact, those above it, and of those equal to it the
    // first ones that make k.  128 rows of 201088 logits, bf16, of which a mask leaves 100: both
    // launches 32 us, by bits as below 1824; without a mask 23.
    __syncthreads();
    if (t == 0) kept = 0;
    bound(std::integral_constant<int, 32>(), 0);
    const int rounds = (units + kPartThreads - 1) / kPartThreads;
    auto unit = [&](Raw& x16, int u) {
      x16.w[0] = *(const u32x4_any*)(x + begin + min(u, units - 1) * kEach);
      return u < units;
    };
#pragma unroll 4
    for (int r = 0; r < rounds; ++r) {
      Raw again;
      const int u = r * kPartThreads + t;
      const bool in = unit(again, u);
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (in && again(e) > least) keep(again(e), begin + u * kEach + e);
    }
    if (t < tail && extra > least) keep(extra, end - tail + t);
    __syncthreads();
    n = kept;
    chosen = n <= kPartList - kMost;
    // (the last round: the numbers behind the units)
    for (int r = 0; chosen && r <= rounds && n < k; ++r) {
      Raw again;
      const int u = r * kPartThreads + t;
      const bool in = r < rounds && unit(again, u);
      int mine = r == rounds && t < tail && extra == least ? 1 : 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) mine += in && again(e) == least ? 1 : 0;
      int upto = mine;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(upto, off, 64);
        upto += lane >= off ? o : 0;
      }
      if (lane == 63) wcount[r & 1][wave] = upto;
      __syncthreads();
      int at = n + upto - mine, all = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        at += w < wave ? wcount[r & 1][w] : 0;
        all += wcount[r & 1][w];
      }
      if (r == rounds && mine && at < k) list[at] = Item{extra, end - tail + t};
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (in && again(e) == least) {
          if (at < k) list[at] = Item{again(e), begin + u * kEach + e};
          ++at;
        }
      n = min(n + all, k);
    }
    __syncthreads();
  }
  if (!chosen) {
    // Too many are above it (a few lanes hold them all): the k-th best by bits, of the images and
    // then of the places among those equal to it, counting the whole stretch each time (from
    // memory: a copy in registers would cost every call a third of its waves).
    auto count = [&](auto which, int turn) {
      int c = 0;
#pragma unroll 1
      for (int p = begin + t; p < end; p += kPartThreads) c += which(image(number(p)), p) ? 1 : 0;
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) c += __shfl_xor(c, off, 64);
      if (lane == 0) wcount[turn & 1][wave] = c;
      __syncthreads();
      c = 0;
      for (int w = 0; w < kWaves; ++w) c += wcount[turn & 1][w];
      return c;
    };
    __syncthreads();
    int turn = 0;
    uint32_t kth = 0u;
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit, ++turn) {
      const uint32_t next = kth | 1u << bit;
      if (count([&](uint32_t y, int) { return y >= next; }, turn) >= k) kth = next;
    }
    int last = begin - 1;  // places up to `last` + 1 of those equal to it
    const int rest = k - count([&](uint32_t y, int) { return y > kth; }, turn++);
#pragma unroll 1
    for (int step = 1 << (31 - __builtin_clz(end - begin)); step; step >>= 1, ++turn)
      if (count([&](uint32_t y, int p) { return y == kth && p <= last + step; }, turn) < rest)
        last += step;
    if (t == 0) wcount[turn & 1][0] = 0;
    __syncthreads();
#pragma unroll 1
    for (int p = begin + t; p < end; p += kPartThreads) {
      const uint32_t y = image(number(p));
      if (y > kth || (y == kth && p <= last + 1)) {  // k of them, in any order
        const int at = atomicAdd(&wcount[turn & 1][0], 1);
        if (at < kPartList)
          list[at] = Item{number(p), p};
      }
    }
    __syncthreads();
    n = min(wcount[turn & 1][0], kPartList);
  }
  rank_all<kPartThreads>(n, ranks, [&](int i) { return list[i]; },
                         [](const Item& a, const Item& b) {
                           return a.x > b.x || (a.x == b.x && a.token < b.token);
                         });
  __syncthreads();
  Item* const out = items + (size_t)blockIdx.x * k;
  for (int i = t; i < n; i += kPartThreads)
    if (ranks[i] < k) out[ranks[i]] = list[i];
  for (int i = n + t; i < k; i += kPartThreads) out[i] = Item{0.f, -1};
}

// One workgroup a request: its rows' sums, then the k best of its lists.
constexpr int kMergeThreads = 1024, kMergeList = kMergeThreads;
// As many are compared with one another at once; us of both launches for 4 beams (k = 8) and for
// 128 (k = 16) of which a mask leaves 3 tokens: up to 128 or 256 25.6 and 39, 512 25.6 and 78, all
// 1024 179 and 78.
constexpr int kMergeFew = 256;
struct Best {
  double v;
  float x;
  int beam, token;
  __device__ __forceinline__ bool before(const Best& o) const {
    if (v != o.v) return v > o.v;
    if (beam != o.beam) return beam < o.beam;
    if (x != o.x) return x > o.x;
    return token < o.token;
  }
};

__global__ __launch_bounds__(kMergeThreads) void merge_kernel(
    const Stat* __restrict__ stats, const Item* __restrict__ items,
    const float* __restrict__ scores, int W, int V, int k, int parts,
    float* __restrict__ out_scores, int* __restrict__ out_beams, int* __restrict__ out_tokens) {
  constexpr int kWaves = kMergeThreads / 64;
  __shared__ double row_m[kMost], row_lse[kMost];  // row_lse NaN: a beam without continuations
  __shared__ float row_score[kMost];
  __shared__ Best list[kMergeList];
  __shared__ int ranks[kMergeList];
  __shared__ uint32_t wbound[kWaves];
  __shared__ uint64_t wexact[kWaves];
  __shared__ uint32_t logit[2];  // of those equal to the bound, from .. to
  __shared__ int found;
  const int r = blockIdx.x, t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const int each = parts * k, total = W * each;
  // the first kHeld candidates of a thread stay in registers, most calls' all; their loads go first
  constexpr int kHeld = 2;
  const Item* const mine = items + (size_t)r * total;
  Item first[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) first[j] = mine[min(t + j * kMergeThreads, total - 1)];
  for (int b = wave; b < W; b += kWaves) {
    const Stat* const st = stats + ((size_t)r * W + b) * parts;
    const float score = scores[(size_t)r * W + b];
    float m = -INFINITY;
    for (int p = lane; p < parts; p += 64) m = fmaxf(m, st[p].m);
    m = wave_max(m);
    double s = 0.0;
    for (int p = lane; p < parts; p += 64) {
      const Stat x = st[p];
      s += x.sum * (x.m == m || x.sum == 0.0 ? 1.0 : exp((double)x.m - (double)m));
    }
    s = moe::wave_sum_f64(s);
    if (lane == 0) {
      const bool good = m > -INFINITY && m < INFINITY && s == s &&
                        score > -INFINITY && score < INFINITY;
      row_m[b] = m;
      row_score[b] = score;
      row_lse[b] = good ? log(s) : __builtin_nan("");
    }
  }
  __syncthreads();
  // candidate i of the request's lists; of a beam without continuations the first k tokens
  auto made = [&](int i, const Item& x, Best& c) {
    const int b = i / each, j = i - b * each;
    const double lse = row_lse[b];
    c.beam = b;
    if (lse != lse) {
      c.v = -INFINITY;
      c.x = -INFINITY;
      c.token = j;
      return j < min(k, V);
    }
    c.x = x.x;
    c.token = x.token;
    c.v = (double)row_score[b] + (((double)x.x - row_m[b]) - lse);
    return x.token >= 0;
  };
  auto candidate = [&](int i, Best& c) { return made(i, mine[i], c); };
  auto high = [](double v) {  // order-preserving image of its upper half
    const uint32_t u = (uint32_t)(__builtin_bit_cast(uint64_t, v + 0.0) >> 32);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
  };
  Best c, held[kHeld];
  uint32_t lm = 0u, image[kHeld];  // 0: none
  const int rest = t + kHeld * kMergeThreads;
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    const int i = t + j * kMergeThreads;
    image[j] = i < total && made(i, first[j], held[j]) ? high(held[j].v) : 0u;
    lm = max(lm, image[j]);
  }
  for (int i = rest; i < total; i += kMergeThreads)
    if (candidate(i, c)) lm = max(lm, high(c.v));
  // (q = 1: beams' scores lie far apart, and one wave may hold all of the best)
  const uint32_t bound = kth_of_lanes<kBoundBits + 3>(lm, k);
  if (lane == 0) wbound[wave] = bound;
  if (t == 0) found = 0;
  ranks[t] = 0;
  __syncthreads();
  const uint32_t top = max(nth_of(wbound, kWaves, 1), 1u);
  auto keep = [&](const Best& x) {
    const int at = atomicAdd(&found, 1);
    if (at < kMergeList) list[at] = x;
  };
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
    if (image[j] >= top) keep(held[j]);
  for (int i = rest; i < total; i += kMergeThreads)
    if (candidate(i, c) && high(c.v) >= top) keep(c);
  __syncthreads();
  int n = found;
  auto write = [&](int rank, const Best& x) {
    out_scores[(size_t)r * k + rank] = (float)x.v;
    out_beams[(size_t)r * k + rank] = x.beam;
    out_tokens[(size_t)r * k + rank] = x.token;
  };
  if (n > kMergeFew) {
    // Many reach the bound (scores equal, as -inf is where a mask leaves few tokens): with it
    // exact, those above it, and of those equal to it the first ones that make k: where
    // their logits are equal too, the lists' order is theirs (beam, stretch, token).
    auto all_bits = [](double v) {
      const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
      return u >> 63 ? ~u : u | (uint64_t)1 << 63;
    };
    uint64_t most = 0u;  // (no number's)
    for (int i = t; i < total; i += kMergeThreads)
      if (candidate(i, c)) most = max(most, all_bits(c.v));
    most = kth_of_lanes<64>(most, k);
    __syncthreads();
    if (t == 0) {
      found = 0;
      logit[0] = ~0u;
      logit[1] = 0u;
    }
    if (lane == 0) wexact[wave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) most = max(most, wexact[w]);
    for (int i = t; i < total; i += kMergeThreads)
      if (candidate(i, c)) {
        const uint64_t u = all_bits(c.v);
        if (u > most) keep(c);
        if (u == most) {
          atomicMin(&logit[0], beam::image(c.x));
          atomicMax(&logit[1], beam::image(c.x));
        }
      }
    __syncthreads();
    n = found;
    if (n < k && logit[0] != logit[1]) n = kMergeList + 1;  // (their own order is wanted)
    for (int i0 = 0; n < k && i0 < total; i0 += 64) {  // (each wave for itself, the first writes)
      const bool is = i0 + lane < total && candidate(i0 + lane, c) && all_bits(c.v) == most;
      const uint64_t who = __ballot(is);
      const int at = n + __builtin_amdgcn_mbcnt_hi(
                             (uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0u));
      if (wave == 0 && is && at < k) list[at] = c;
      n = min(n + (int)__popcll(who), k);
    }
    __syncthreads();
  }
  if (n <= kMergeList) {
    rank_all<kMergeThreads>(n, ranks, [&](int i) { return list[i]; },
                            [](const Best& x, const Best& y) { return x.before(y); });
    __syncthreads();
    for (int i = t; i < n; i += kMergeThreads)
      if (ranks[i] < k) write(ranks[i], list[i]);
    return;
  }
  // Too many: one after the other, each the best of those behind the last
  Best last{INFINITY, INFINITY, -1, -1};
  const Best none{-INFINITY, -INFINITY, INT32_MAX, INT32_MAX};
  for (int rank = 0; rank < k; ++rank) {
    Best best = none;
    for (int i = t; i < total; i += kMergeThreads)
      if (candidate(i, c) && last.before(c) && c.before(best)) best = c;
    __syncthreads();
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      const Best o{__shfl_xor(best.v, off, 64), __shfl_xor(best.x, off, 64),
                   __shfl_xor(best.beam, off, 64), __shfl_xor(best.token, off, 64)};
      if (o.before(best)) best = o;
    }
    if (lane == 0) list[wave] = best;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w)
      if (list[w].before(best)) best = list[w];
    last = best;
    if (t == 0) write(rank, best);
  }
}

// Chunks of a stretch: as many as leave 512 workgroups, two a CU, of a call's rows.  16 requests of
// 8 beams of 201088 logits, us of both launches: 256 workgroups 34, 512 25, 1024 29 (more lists for
// the second one).
inline int chunks_of(int64_t rows, int vocab) {
  const int64_t all = ((int64_t)vocab + kChunk - 1) / kChunk;
  const int64_t parts = std::min(all, std::max<int64_t>(1, (512 + rows - 1) / rows));
  return (int)((all + parts - 1) / parts);
}
inline int64_t parts_of(int64_t rows, int vocab) {
  const int64_t each = (int64_t)chunks_of(rows, vocab) * kChunk;
  return (vocab + each - 1) / each;
}
inline size_t round256(size_t x) { return (x + 255) / 256 * 256; }

}  // namespace beam

extern "C" {

// 0 where there are too many stretches for a launch
size_t attn_beam_state_bytes(int64_t rows, int vocab, int k) {
  const int64_t n = rows * beam::parts_of(rows, vocab);
  if (n * k >= (int64_t)1 << 31 || n * beam::kPartThreads >= (int64_t)1 << 32) return 0;
  return beam::round256(n * sizeof(beam::Stat)) + n * k * sizeof(beam::Item);
}

int attn_launch_beam(const void* logits, bool f32, const float* scores, int batch, int width,
                     int vocab, int k, float* out_scores, int* out_beams, int* out_tokens,
                     void* state, hipStream_t s) {
  const int64_t rows = (int64_t)batch * width;
  const int parts = (int)beam::parts_of(rows, vocab), chunks = beam::chunks_of(rows, vocab);
  beam::Stat* stats = (beam::Stat*)state;
  beam::Item* items =
      (beam::Item*)((char*)state + beam::round256(rows * parts * sizeof(beam::Stat)));
  const dim3 grid((unsigned)(rows * parts)), threads(beam::kPartThreads);
  if (f32)
    hipLaunchKernelGGL(beam::part_kernel<float>, grid, threads, 0, s, (const float*)logits, vocab,
                       k, parts, chunks, stats, items);
  else
    hipLaunchKernelGGL(beam::part_kernel<uint16_t>, grid, threads, 0, s, (const uint16_t*)logits,
                       vocab, k, parts, chunks, stats, items);
  if (hipGetLastError() != hipSuccess) return -6;
  hipLaunchKernelGGL(beam::merge_kernel, dim3(batch), dim3(beam::kMergeThreads), 0, s, stats,
                     items, scores, width, vocab, k, parts, out_scores, out_beams, out_tokens);
  return hipGetLastError() == hipSuccess ? 0 : -6;
}

}  // extern "C"
