// The 8-bit paged KV cache (gfx950): rows of a bf16 cache put into it, rows read
// back, and the attention of decode and of chunks of new tokens over it.  The
// format and its page layout: attn_common.h.  (The QKV epilogue that appends to
// it is qkv_rope_append_kernel<true> of attn_kernels.hip.)
#include <type_traits>

#include "attn_common.h"

namespace attn {

constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------------------
// Rows of a bf16 cache (by slot) quantised into the 8-bit cache, and rows read back.
// Bound by their bytes.  A wave takes four tokens' runs; lane (k or v, head, quarter of
// 16 dims).  A wave a token, v's codes moved byte by byte, had 49 us for 40960 rows read
// where runs have 23.6, and 5.4 us for 1000 where they have 5.6.  40960 rows are
// quantised in 31 us (4.1 TB/s).  (The 23.6 us, 5.4 TB/s, are of passes over three caches of
// 43 MB into one output of 84 MB, which the last-level cache holds between them; a copy
// of 2 GB reaches 4.95.)

template <int kRun>
__device__ __forceinline__ void quantize_run(const uint8_t* __restrict__ src, int src_pages,
                                             const int* __restrict__ src_slots,
                                             uint8_t* __restrict__ cache, int num_pages,
                                             int slot) {
  const int lane = threadIdx.x & 63, kv = lane >> 5, hk = (lane >> 2) & 7, part = lane & 3;
  u32x4 a[kRun], b[kRun], codes[kRun];
  uint32_t s[kRun];
  bool good[kRun], all = true;
#pragma unroll
  for (int t = 0; t < kRun; ++t) {
    const int from = src_slots[t];
    good[t] = from >= 0 && from < src_pages * kPage;
    all = all && good[t];
    const int at = good[t] ? from : 0;
    const uint8_t* row = src + ((((size_t)(at / kPage) * 2 + kv) * kHkv + hk) * kPage +
                                at % kPage) * (kD * 2) + part * 32;
    a[t] = *(const u32x4*)row;
    b[t] = *(const u32x4*)(row + 16);
  }
#pragma unroll
  for (int t = 0; t < kRun; ++t) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      top = max(max(top, a[t][j] & 0x7FFFu), (a[t][j] >> 16) & 0x7FFFu);
      top = max(max(top, b[t][j] & 0x7FFFu), (b[t][j] >> 16) & 0x7FFFu);
    }
    s[t] = fp8_scale_of(quad_max(top));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      codes[t][j] = j < 2 ? fp8_codes(a[t][2 * j], a[t][2 * j + 1], s[t], kv)
                          : fp8_codes(b[t][2 * j - 4], b[t][2 * j - 3], s[t], kv);
  }
  uint8_t* const page = fp8_page(cache, slot, num_pages);
  const int token = slot % kPage;
  if (kRun == 4 && all) {
    if (kv == 0) {
#pragma unroll
      for (int t = 0; t < kRun; ++t)
        *(u32x4*)(page + hk * kFp8Head + (token + t) * kFp8Row + part * 16) = codes[t];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t w[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) w[t] = codes[t % kRun][j];
        transpose4(w);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(uint32_t*)(page + fp8_v_at(hk, token, part * 16 + 4 * j + i)) = w[i];
      }
    }
    if (part == 0) {
      uint32_t scales = 0;
#pragma unroll
      for (int t = 0; t < kRun; ++t) scales |= s[t] << (8 * t);
      *(uint32_t*)(page + fp8_scale_at(hk, kv, token)) = scales;
    }
    return;
  }
#pragma unroll
  for (int t = 0; t < kRun; ++t) {
    if (!good[t]) continue;
    if (kv == 0) {
      *(u32x4*)(page + hk * kFp8Head + (token + t) * kFp8Row + part * 16) = codes[t];
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        page[fp8_v_at(hk, token + t, part * 16 + j)] =
            (uint8_t)(codes[t][j >> 2] >> (8 * (j & 3)));
    }
    if (part == 0) page[fp8_scale_at(hk, kv, token + t)] = (uint8_t)s[t];
  }
}

__global__ __launch_bounds__(256) void fp8_quantize_kernel(
    const uint8_t* __restrict__ src, int src_pages, const int* __restrict__ src_slots, int n,
    uint8_t* __restrict__ cache, int num_pages, const int* __restrict__ slots) {
  const int wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int first = wave * 4;
  if (first >= n) return;
  const SlotRuns runs(slots, first, n);
  for (int t = 0; t < 4 && first + t < n; ++t) {
    if (!(runs.begins >> t & 1)) continue;
    const int i = first + t, length = runs.length(t);
    if (fp8_quad(slots[i], length, num_pages))
      quantize_run<4>(src, src_pages, src_slots + i, cache, num_pages, slots[i]);
    else
      for (int j = i; j < i + length; ++j)
        if (fp8_page(cache, slots[j], num_pages))
          quantize_run<1>(src, src_pages, src_slots + j, cache, num_pages, slots[j]);
  }
}

// Back to bf16, k and v [n, 8, 64]: exact (a code has four significant bits, and no
// value is below bf16's normal range); a row of scale 255 gives NaN, a slot outside
// the pool zeros.
template <int kRun>
__device__ __forceinline__ void read_run(const uint8_t* __restrict__ cache, int num_pages,
                                         int slot, int i, uint16_t* __restrict__ k_out,
                                         uint16_t* __restrict__ v_out) {
  const int lane = threadIdx.x & 63, kv = lane >> 5, hk = (lane >> 2) & 7, part = lane & 3;
  const uint8_t* const page = fp8_page(const_cast<uint8_t*>(cache), slot, num_pages);
  const int token = slot % kPage;
  u32x4 codes[kRun] = {};
  uint32_t s[kRun];
#pragma unroll
  for (int t = 0; t < kRun; ++t) s[t] = kFp8MinScale;
  if (page) {
    uint32_t scales;
    if (kRun == 4)
      scales = *(const uint32_t*)(page + fp8_scale_at(hk, kv, token));
    else
      scales = page[fp8_scale_at(hk, kv, token)];
    if (kv == 0) {
#pragma unroll
      for (int t = 0; t < kRun; ++t)
        codes[t] = *(const u32x4*)(page + hk * kFp8Head + (token + t) * kFp8Row + part * 16);
    } else if (kRun == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = *(const uint32_t*)(page + fp8_v_at(hk, token, part * 16 + 4 * j + i));
        transpose4(w);
#pragma unroll
        for (int t = 0; t < kRun; ++t) codes[t][j] = w[t];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        codes[0][j >> 2] |= (uint32_t)page[fp8_v_at(hk, token, part * 16 + j)] << (8 * (j & 3));
    }
#pragma unroll
    for (int t = 0; t < kRun; ++t) s[t] = (scales >> (8 * t)) & 255u;
  }
  uint16_t* const dst = (kv ? v_out : k_out) + ((size_t)i * kHkv + hk) * kD + part * 16;
#pragma unroll
  for (int t = 0; t < kRun; ++t) {
    const float scale = __uint_as_float(min(s[t], kFp8BadScale - 1u) << 23);
    u32x4 lo = __builtin_bit_cast(u32x4, fp8_to_bf16(codes[t][0], codes[t][1], scale));
    u32x4 hi = __builtin_bit_cast(u32x4, fp8_to_bf16(codes[t][2], codes[t][3], scale));
    if (s[t] == kFp8BadScale) lo = hi = u32x4{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
    *(u32x4*)(dst + t * kHkv * kD) = lo;
    *(u32x4*)(dst + t * kHkv * kD + 8) = hi;
  }
}

__global__ __launch_bounds__(256) void fp8_read_kernel(const uint8_t* __restrict__ cache,
                                                       int num_pages,
                                                       const int* __restrict__ slots, int n,
                                                       uint16_t* __restrict__ k_out,
                                                       uint16_t* __restrict__ v_out) {
  const int wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int first = wave * 4;
  if (first >= n) return;
  const SlotRuns runs(slots, first, n);
  for (int t = 0; t < 4 && first + t < n; ++t) {
    if (!(runs.begins >> t & 1)) continue;
    const int i = first + t, length = runs.length(t);
    if (fp8_quad(slots[i], length, num_pages))
      read_run<4>(cache, num_pages, slots[i], i, k_out, v_out);
    else
      for (int j = i; j < i + length; ++j)
        read_run<1>(cache, num_pages, slots[j], j, k_out, v_out);
  }
}

// ---------------------------------------------------------------------------
// Attention.  For a query at position p of a sequence and the keys j <= p (and
// > p - window, where there is one):
//   out = sum_j p_j v_j / (sum_j p_j + exp(sink)),  p_j = exp(sm_scale q . k_j)
// rounded to bf16 once.  (The bf16 cache's form rounds o, the sink's factor and
// their product, as the operators it restates do.)  A query that sees no key gets
// 0.  Scores, maxima, sums and outputs in fp32; exponents in units of log2.

// o over the sum and the sink's share, at the reference point m (log2).  l is 0
// only where no key was seen (m is a key's score, so its p is 1).
__device__ __forceinline__ float sink_share(float l, float m, uint16_t sink) {
  return l == 0.0f ? 0.0f : 1.0f / (l + __builtin_amdgcn_exp2f(fmaf(bf2f(sink), kLog2e, -m)));
}

// How many splits a tile's `blocks` blocks of 64 keys are shared out over: as many as
// have `least` blocks, more than 32 only where they have 16, at most `most`.  It follows
// from the keys and not from the caller's bound on them, which only trims the grid.
constexpr int kFp8Block = 64;
constexpr float kFp8Most = 16777216.0f;  // 2^24
struct Shares {
  int each, used;  // blocks of a split, splits with any
  __device__ __forceinline__ Shares(int blocks, int most, int least) {
    const int n = min(min(most, (blocks + least - 1) / least), max(32, (blocks + 15) / 16));
    each = n > 0 ? (blocks + n - 1) / n : 0;
    used = each > 0 ? (blocks + each - 1) / each : 0;
  }
};

// The keys that a tile's tokens see: positions lo .. last (none if last < lo).
struct Sight {
  int lo, last, first, blocks;  // first block of 64, number of blocks
  __device__ __forceinline__ Sight(int pos, int tokens, int window) {
    lo = window > 0 && pos >= window ? pos - window + 1 : 0;
    last = pos + tokens - 1;
    first = lo / kFp8Block;
    blocks = last >= lo ? last / kFp8Block - first + 1 : 0;
  }
};

struct RowsArgs {
  const uint16_t* q;
  const int* q_indptr;  // chunks
  const uint8_t* cache;
  const int* page_indptr;
  const int* page_indices;
  const int* kv_len;
  const uint16_t* sinks;
  uint16_t* out;
  float* part_o;   // [splits][rows][64][64], rows: sequences, or a chunk's tiles' tokens
  float* part_ml;  // [splits][rows][64][2]
  int* arrive;     // decode: [batch][8], left zero
  int64_t max_span;
  int num_pages, window, splits, least, rows, tiles;
  float c2;        // sm_scale log2(e)
};

// Decode: one token a sequence.  Bound by the cache's bytes, so nothing but loads is on
// the way: a wave takes blocks of 64 keys (four pages) alone, from global memory to
// registers, no LDS and no barrier before the end; a load takes the 1 KB that a page
// holds of a kv head's k or v, past the caches (nontemporal: read once; 7.1 TB/s
// against 6.3 in a kernel that only loads).  Both products run on
// v_mfma_f32_16x16x32_bf16 with the 8 heads of a kv head in columns 0 .. 7 and again
// in 8 .. 15:
//  * S^T = K Q^T: row r of a page's score tile is its key r, so lane (r, g) loads dims
//    16 g .. 16 g + 15 of it, and result element i of lane (column, g) is key 4 g + i;
//  * O^T = V^T P^T over two pages: the lane's P operand then is its own scores, slot
//    4 kk + i for page kk of the two; V^T's slots the same keys, dims 16 dt + r, as the
//    cache holds them.
// Columns 0 .. 7 keep the scores of the block's first two pages and 8 .. 15 those of
// the others, each column with a softmax state of its own, so that every lane's
// exponential is of use; each half's products give one half of the columns, the other
// is not looked at.
// Codes go to bf16 exactly (k with its scale, whose row a lane holds alone; v
// without: its scales multiply p); pv enters as two bf16 pieces, about 16 bits.
// k of the next block is in flight from the scores on, v from the products on.
// 64 sequences of 1024 to 4096 keys 36 us (158 MB, 4.4 TB/s), two of up to 131072 44 us (4.8
// TB/s), one of 777 6.8 us.
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4))) void fp8_decode_kernel(
    RowsArgs a) {
  constexpr int kStates = 8;  // of a head in a workgroup: 4 waves, two halves
  __shared__ __align__(16) float obuf[4][16][kD + 4];
  __shared__ float mbuf[4][16], lbuf[4][16];
  // x: (sequence, kv head), y: split
  const int hk = blockIdx.x % kHkv, b = blockIdx.x / kHkv, share = blockIdx.y;
  const int L = a.kv_len[b], pos = L - 1;
  const Sight sight(pos, 1, a.window);
  const Shares shares(sight.blocks, a.splits, a.least);
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int lane = t & 63, r = lane & 15, g = lane >> 4;
  const bool second = r >= 8;
  const bool too_long = (int64_t)sight.last + 1 - sight.lo > a.max_span;
  if (share >= max(shares.used, 1) || (too_long && share > 0)) return;
  if (too_long) {
    for (int i = t; i < kGroup * kD; i += 256)
      a.out[((size_t)b * kHq + hk * kGroup) * kD + i] = 0x7FC0;
    return;
  }
  const PageList pages{a.page_indices + a.page_indptr[b],
                       a.page_indptr[b + 1] - a.page_indptr[b], a.num_pages};
  const int last_page = max(0, min(pages.count - 1, (L - 1) / kPage));
  const int begin = share * shares.each, end = min(begin + shares.each, sight.blocks);
  const unsigned reach = a.window > 0 ? a.window : 0x7FFFFFFFu;  // keys back that it sees

  // The wave's blocks: begin + wave, + 4, ...  Lane 4 j + p holds the page p of the
  // j-th of 16 blocks.
  int ids = 0;
  auto fetch_ids = [&](int blk) {
    const int i = (sight.first + blk + 4 * (lane >> 2)) * 4 + (lane & 3);
    ids = pages.count > 0 ? pages.clamp(pages.ids[min(i, last_page)]) : 0;
  };
  u32x4 k[4], v[4];      // of the block's pages
  uint32_t ks[4], vs[2];  // k's scale of key r; v's of keys 4 g .. of the lane's own pages
  const unsigned k_at = hk * kFp8Head + r * kFp8Row + g * 16;
  const unsigned v_at = kFp8V + hk * kFp8Head + lane * 16;
  const unsigned s_at = kFp8Scales + hk * 2 * kPage;
  auto page_of = [&](int j, int p) {  // of the j-th block at hand
    return a.cache + (size_t)(unsigned)__builtin_amdgcn_readlane(ids, 4 * j + p) * kFp8Page;
  };
  auto load_k = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint8_t* page = page_of(j, p);
      k[p] = __builtin_nontemporal_load((const u32x4*)(page + k_at));
      ks[p] = page[s_at + r];
    }
  };
  auto load_v = [&](int j) __attribute__((always_inline)) {
    const uint8_t* page[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      page[p] = page_of(j, p);
      v[p] = __builtin_nontemporal_load((const u32x4*)(page[p] + v_at));
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
      vs[kk] = *(const uint32_t*)((second ? page[2 + kk] : page[kk]) + s_at + kPage + 4 * g);
  };
  fetch_ids(begin + wave);

  // Q operand: column r is head r % 8
  bf16x8 qv[2];
  {
    const u32x4* src = (const u32x4*)(a.q + ((size_t)b * kHq + hk * kGroup + (r & 7)) * kD);
    qv[0] = moe::as_bf16x8(src[2 * g]);
    qv[1] = moe::as_bf16x8(src[2 * g + 1]);
  }
  f32x4 o[2][4];
  float mneg = INFINITY, l = 0.f;  // minus the column's reference point (not set: inf)
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) o[x][dt] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int c0 = begin + wave; c0 < end; c0 += 64) {  // 16 of the wave's blocks
    if (c0 != begin + wave) fetch_ids(c0);
    const int n = min(16, (end - c0 + 3) / 4);
    load_k(0);
    load_v(0);
    for (int j = 0; j < n; ++j) {
      const int kb = (sight.first + c0 + 4 * j) * kFp8Block;
      f32x4 st[2];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        f32x4 s[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const u32x4 kp = k[2 * x + kk];
          const float scale = __uint_as_float(min(ks[2 * x + kk], kFp8BadScale - 1u) << 23);
          s[x] = mfma_bf16(fp8_to_bf16(kp[0], kp[1], scale), qv[0], f32x4{0.f, 0.f, 0.f, 0.f});
          s[x] = mfma_bf16(fp8_to_bf16(kp[2], kp[3], scale), qv[1], s[x]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) st[kk][i] = second ? s[1][i] : s[0][i];
      }
      if (j + 1 < n) load_k(j + 1);
      // every key of the block is seen
      const bool whole = kb + kFp8Block - 1 <= pos && (a.window <= 0 || kb > pos - a.window);
      const int back = pos - (kb + (second ? 32 : 0) + 4 * g);  // of the lane's first key
      if (!whole) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            st[kk][i] = (unsigned)(back - 16 * kk - i) < reach ? st[kk][i] : -INFINITY;
      }
      float p[8], ps;
      auto exps = [&](float mn) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          p[i] = __builtin_amdgcn_exp2f(fmaf(st[i >> 2][i & 3], a.c2, mn));
        ps = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      };
      exps(mneg);
      if (__any(!(ps < kFp8Most))) {
        float mx = st[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, st[i >> 2][i & 3]);
        const float mo = -mneg, mn = fmaxf(mo, group_max(mx) * a.c2);
        const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mo - mn);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[x][dt][i] *= alpha;
        l *= alpha;
        mneg = -mn;
        exps(mn == -INFINITY ? 0.0f : -mn);
      }
      l += ps;
      bf16x8 ph, pl;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // times v's scale.  A bad row's byte gives an infinite factor: NaN from its
          // codes 0; a hidden key's p of 0 stays 0
          float pv = p[4 * kk + i] * __uint_as_float(((vs[kk] >> (8 * i)) & 255u) << 23);
          if (!whole) pv = (unsigned)(back - 16 * kk - i) < reach ? pv : 0.0f;
          const __bf16 hi = (__bf16)pv;
          ph[4 * kk + i] = hi;
          pl[4 * kk + i] = (__bf16)(pv - (float)hi);
        }
      if (kb + kFp8Block > L) {  // stale codes past the sequence's end may be NaN
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const int left = min(max(L - (kb + 16 * p + 4 * g), 0), 4);
          const uint32_t keep = left == 4 ? ~0u : (1u << (8 * left)) - 1u;
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) v[p][dt] &= keep;
        }
      }
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const bf16x8 va = fp8_to_bf16(v[2 * x][dt], v[2 * x + 1][dt], 1.0f);
          o[x][dt] = mfma_bf16(va, ph, o[x][dt]);
          o[x][dt] = mfma_bf16(va, pl, o[x][dt]);
        }
      if (j + 1 < n) load_v(j + 1);
    }
  }

  // The eight states of a head merged, in a fixed order: 32 threads a head, two
  // dimensions each
  l += __shfl_xor(l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);
  if (g == 0) {
    mbuf[wave][r] = -mneg;
    lbuf[wave][r] = l;
  }
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) {
    f32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = second ? o[1][dt][i] : o[0][dt][i];
    *(f32x4*)&obuf[wave][r][16 * dt + 4 * g] = w;
  }
  __syncthreads();
  const int h = t >> 5, i0 = t & 31, d = 2 * i0;
  // the weight of a state; one that saw no key: m = -inf, l = 0, o = 0
  auto weight = [](float m, float l, float top) {
    return m == -INFINITY && l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - top);
  };
  float mt = -INFINITY, lt = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
  for (int s = 0; s < kStates; ++s) mt = fmaxf(mt, mbuf[s >> 1][h + 8 * (s & 1)]);
#pragma unroll
  for (int s = 0; s < kStates; ++s) {
    const int w = s >> 1, c = h + 8 * (s & 1);
    const float wgt = weight(mbuf[w][c], lbuf[w][c], mt);
    lt = fmaf(lbuf[w][c], wgt, lt);
    const float2 ow = *(const float2*)&obuf[w][c][d];
    o0 = fmaf(ow.x, wgt, o0);
    o1 = fmaf(ow.y, wgt, o1);
  }
  const size_t at = (size_t)b * kHq + hk * kGroup + h, step = (size_t)a.rows * kHq;
  const uint16_t sink = a.sinks[hk * kGroup + h];
  auto write = [&](float l_all, float m_all) {
    const float f = sink_share(l_all, m_all, sink);
    *(uint32_t*)(a.out + at * kD + d) = (uint32_t)f2bf(o0 * f) | ((uint32_t)f2bf(o1 * f) << 16);
  };
  const int used = shares.used;
  if (used <= 1) {
    write(lt, mt);
    return;
  }
  // to be merged by a workgroup of this launch: device scope
  const size_t pt = at + (size_t)share * step;
  store_dev((uint64_t*)(a.part_o + pt * kD + d),
            (uint64_t)__float_as_uint(o0) | ((uint64_t)__float_as_uint(o1) << 32));
  if (i0 == 0)
    store_dev((uint64_t*)(a.part_ml + pt * 2),
              (uint64_t)__float_as_uint(mt) | ((uint64_t)__float_as_uint(lt) << 32));
  // The last of the head group's splits to finish merges them: its stores are
  // done (vmcnt), the workgroup meets, one thread counts; the one that completes
  // the count leaves it zero for the next call.
  __shared__ int is_last;
  moe::wait_vmcnt<0>();
  __syncthreads();
  if (t == 0) {
    int* cnt = a.arrive + b * kHkv + hk;
    const int prev = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    is_last = prev == used - 1;
    if (is_last) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!is_last) return;
  // The states (a lane a split, its weights to LDS) and o (a thread two dimensions, over the
  // splits in order, sixteen loads in flight, the first beside the states').
  __shared__ float wgt[kGroup][64];  // used <= 64
  float ms[2], ls[2];
  mt = -INFINITY;
  lt = o0 = o1 = 0.f;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int s = i0 + 32 * j;
    uint64_t ml = (uint64_t)0xFF800000u;  // m = -inf, l = 0
    if (s < used) ml = load_dev((const uint64_t*)(a.part_ml + (at + s * step) * 2));
    ms[j] = __uint_as_float((uint32_t)ml);
    ls[j] = __uint_as_float((uint32_t)(ml >> 32));
  }
  for (int s0 = 0; s0 < used; s0 += 16) {
    uint64_t po[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      po[i] = load_dev((const uint64_t*)(a.part_o + (at + min(s0 + i, used - 1) * step) * kD + d));
    if (s0 == 0) {
      mt = fmaxf(ms[0], ms[1]);
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) mt = fmaxf(mt, __shfl_xor(mt, off, kWave));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float w = weight(ms[j], ls[j], mt);
        if (i0 + 32 * j < used) wgt[h][i0 + 32 * j] = w;
        lt = fmaf(ls[j], w, lt);
      }
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) lt += __shfl_xor(lt, off, kWave);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (s0 + i < used) {
        o0 = fmaf(__uint_as_float((uint32_t)po[i]), wgt[h][s0 + i], o0);
        o1 = fmaf(__uint_as_float((uint32_t)(po[i] >> 32)), wgt[h][s0 + i], o1);
      }
  }
  write(lt, mt);
}

// Chunks of few tokens (drafts under verification): a tile of 2 kCt tokens in kCt tiles
// of 16 columns (token, head), by decode's loads and products, p in two bf16 pieces as
// there: a token gets the same weights whether it is decoded or verified.  (One bf16
// rounding of p, whatever p's sum takes, is 6 to 10% faster: 16 sequences of 5 tokens over
// up to 4000 keys 25.5 us; its errors against 64 bits 0.0020 to 0.0022 where decode's
// and this form's are 0.0017.)  More tokens take more such tiles, which read the
// keys again.  Bound by a wave's own instructions over its blocks: the 16 sequences
// of 5 tokens take 31.8 us in tiles of 4, 27.1 in tiles of 2 (one tile of 8, whose four
// column tiles a wave spill, took twice as long).
template <int kCt>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void fp8_rows_kernel(
    RowsArgs a) {
  constexpr int kCols = 16 * kCt;
  __shared__ __align__(16) float obuf[4][16][kD + 4];  // one column tile of each wave
  __shared__ float mbuf[4][kCols], lbuf[4][kCols];
  // x: (sequence, tile, kv head), y: split
  const int hk = blockIdx.x % kHkv, share = blockIdx.y;
  const int b = blockIdx.x / kHkv / a.tiles, tile = blockIdx.x / kHkv % a.tiles;
  const int qb = a.q_indptr[b], qn = a.q_indptr[b + 1] - qb;
  const int t0 = tile * 2 * kCt;
  if (t0 >= qn) return;
  const int nt = min(2 * kCt, qn - t0);
  const int L = a.kv_len[b], pos = L - qn + t0;  // of the tile's first token
  const Sight sight(pos, nt, a.window);
  const Shares shares(sight.blocks, a.splits, a.least);
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int lane = t & 63, r = lane & 15, g = lane >> 4;
  const int row0 = qb + t0;
  if (share >= max(shares.used, 1)) return;
  const PageList pages{a.page_indices + a.page_indptr[b],
                       a.page_indptr[b + 1] - a.page_indptr[b], a.num_pages};
  const int last_page = max(0, min(pages.count - 1, (L - 1) / kPage));
  const int begin = share * shares.each, end = min(begin + shares.each, sight.blocks);

  // Q operand of column tile ct: column r is token 2 ct + r / 8, head r % 8
  bf16x8 qv[kCt][2];
#pragma unroll
  for (int ct = 0; ct < kCt; ++ct) {
    const int row = row0 + min(2 * ct + (r >> 3), nt - 1);
    const u32x4* src = (const u32x4*)(a.q + ((size_t)row * kHq + hk * kGroup + (r & 7)) * kD);
    qv[ct][0] = moe::as_bf16x8(src[2 * g]);
    qv[ct][1] = moe::as_bf16x8(src[2 * g + 1]);
  }
  const unsigned reach = a.window > 0 ? a.window : 0x7FFFFFFFu;
  f32x4 o[kCt][4];
  float mneg[kCt], l[kCt];  // minus the columns' reference points (not set: inf)
#pragma unroll
  for (int ct = 0; ct < kCt; ++ct) {
    mneg[ct] = INFINITY;
    l[ct] = 0.f;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) o[ct][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // The wave's blocks: begin + wave, + 4, ...  Lane 4 j + p holds the page p of the
  // j-th of 16 blocks.
  int ids = 0;
  auto fetch_ids = [&](int blk) {
    const int i = (sight.first + blk + 4 * (lane >> 2)) * 4 + (lane & 3);
    ids = pages.count > 0 ? pages.clamp(pages.ids[min(i, last_page)]) : 0;
  };
  u32x4 k[4], v[4];       // of the block's pages
  uint32_t ks[4], vs[4];  // k's scale of key r; v's of keys 4 g ..
  const unsigned k_at = hk * kFp8Head + r * kFp8Row + g * 16;
  const unsigned v_at = kFp8V + hk * kFp8Head + lane * 16;
  const unsigned s_at = kFp8Scales + hk * 2 * kPage;
  auto page_of = [&](int j, int p) {  // of the j-th block at hand
    return a.cache + (size_t)(unsigned)__builtin_amdgcn_readlane(ids, 4 * j + p) * kFp8Page;
  };
  auto load_k = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint8_t* page = page_of(j, p);
      k[p] = __builtin_nontemporal_load((const u32x4*)(page + k_at));
      ks[p] = page[s_at + r];
    }
  };
  auto load_v = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint8_t* page = page_of(j, p);
      v[p] = __builtin_nontemporal_load((const u32x4*)(page + v_at));
      vs[p] = *(const uint32_t*)(page + s_at + kPage + 4 * g);
    }
  };
  auto block = [&](int kb, int next) __attribute__((always_inline)) {  // kb: its first key
    bf16x8 ka[4][2];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const float scale = __uint_as_float(min(ks[p], kFp8BadScale - 1u) << 23);
      ka[p][0] = fp8_to_bf16(k[p][0], k[p][1], scale);
      ka[p][1] = fp8_to_bf16(k[p][2], k[p][3], scale);
    }
    if (next >= 0) load_k(next);  // in flight during the rest
    // every token of the tile sees the whole block
    const bool whole = kb + kFp8Block - 1 <= pos && (a.window <= 0 || kb > sight.last - a.window);
    bf16x8 ph[kCt][2], pl[kCt][2];
#pragma unroll
    for (int ct = 0; ct < kCt; ++ct) {
      f32x4 st[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        st[p] = mfma_bf16(ka[p][0], qv[ct][0], f32x4{0.f, 0.f, 0.f, 0.f});
        st[p] = mfma_bf16(ka[p][1], qv[ct][1], st[p]);
      }
      // the token's position behind the lane's first key; it sees `reach` keys back
      const int back = pos + min(2 * ct + (r >> 3), nt - 1) - (kb + 4 * g);
      if (!whole) {
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            st[p][i] = (unsigned)(back - 16 * p - i) < reach ? st[p][i] : -INFINITY;
      }
      f32x4 e[4];
      float ps;
      auto exps = [&](float mn) __attribute__((always_inline)) {
        ps = 0.f;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
#pragma unroll
          for (int i = 0; i < 4; ++i) e[p][i] = __builtin_amdgcn_exp2f(fmaf(st[p][i], a.c2, mn));
          ps += (e[p][0] + e[p][1]) + (e[p][2] + e[p][3]);
        }
      };
      exps(mneg[ct]);
      if (__any(!(ps < kFp8Most))) {
        float mx = -INFINITY;
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, st[p][i]);
        const float mo = -mneg[ct], mn = fmaxf(mo, group_max(mx) * a.c2);
        const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mo - mn);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[ct][dt][i] *= alpha;
        l[ct] *= alpha;
        mneg[ct] = -mn;
        exps(mn == -INFINITY ? 0.0f : -mn);
      }
      l[ct] += ps;
      // times v's scales.  A bad row's byte gives an infinite factor: NaN from its
      // codes 0; a hidden key's p of 0 stays 0
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float pv = e[p][i] * __uint_as_float(((vs[p] >> (8 * i)) & 255u) << 23);
          if (!whole) pv = (unsigned)(back - 16 * p - i) < reach ? pv : 0.0f;
          const __bf16 hi = (__bf16)pv;
          ph[ct][p >> 1][4 * (p & 1) + i] = hi;
          pl[ct][p >> 1][4 * (p & 1) + i] = (__bf16)(pv - (float)hi);
        }
    }
    if (kb + kFp8Block > L) {  // stale codes past the sequence's end may be NaN
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int left = min(max(L - (kb + 16 * p + 4 * g), 0), 4);
        const uint32_t keep = left == 4 ? ~0u : (1u << (8 * left)) - 1u;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) v[p][dt] &= keep;
      }
    }
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      const bf16x8 v0 = fp8_to_bf16(v[0][dt], v[1][dt], 1.0f);
      const bf16x8 v1 = fp8_to_bf16(v[2][dt], v[3][dt], 1.0f);
#pragma unroll
      for (int ct = 0; ct < kCt; ++ct) {
        o[ct][dt] = mfma_bf16(v0, ph[ct][0], o[ct][dt]);
        o[ct][dt] = mfma_bf16(v0, pl[ct][0], o[ct][dt]);
        o[ct][dt] = mfma_bf16(v1, ph[ct][1], o[ct][dt]);
        o[ct][dt] = mfma_bf16(v1, pl[ct][1], o[ct][dt]);
      }
    }
    if (next >= 0) load_v(next);
  };

  for (int c0 = begin + wave; c0 < end; c0 += 64) {  // 16 of the wave's blocks
    fetch_ids(c0);
    const int n = min(16, (end - c0 + 3) / 4);
    load_k(0);
    load_v(0);
    for (int j = 0; j < n; ++j)
      block((sight.first + c0 + 4 * j) * kFp8Block, j + 1 < n ? j + 1 : -1);
  }

  // The four waves' states merged, in wave order
#pragma unroll
  for (int ct = 0; ct < kCt; ++ct) {
    float lt = l[ct];
    lt += __shfl_xor(lt, 16, kWave);
    lt += __shfl_xor(lt, 32, kWave);
    if (g == 0) {
      mbuf[wave][16 * ct + r] = -mneg[ct];
      lbuf[wave][16 * ct + r] = lt;
    }
  }
  const bool alone = shares.used <= 1;
#pragma unroll
  for (int ct = 0; ct < kCt; ++ct) {
    __syncthreads();  // the maxima are there; the last tile's o was read
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) *(f32x4*)&obuf[wave][r][16 * dt + 4 * g] = o[ct][dt];
    __syncthreads();
    const int col = t >> 4, d = (t & 15) * 4, cc = 16 * ct + col;
    const int token = 2 * ct + (col >> 3), head = hk * kGroup + (col & 7);
    if (token >= nt) continue;
    float mt = -INFINITY, lt = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mt = fmaxf(mt, mbuf[w][cc]);
    f32x4 ot = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      // a wave that saw none of the column's keys: m = -inf, l = 0, o = 0
      const float wgt = mbuf[w][cc] == -INFINITY && lbuf[w][cc] == 0.0f
                            ? 0.0f : __builtin_amdgcn_exp2f(mbuf[w][cc] - mt);
      lt = fmaf(lbuf[w][cc], wgt, lt);
#pragma unroll
      for (int i = 0; i < 4; ++i) ot[i] = fmaf(obuf[w][col][d + i], wgt, ot[i]);
    }
    const size_t at = (size_t)(row0 + token) * kHq + head;
    if (alone) {
      const float f = sink_share(lt, mt, a.sinks[head]);
      uint16_t v4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v4[i] = f2bf(ot[i] * f);
      *(uint2*)(a.out + at * kD + d) = make_uint2((uint32_t)v4[0] | ((uint32_t)v4[1] << 16),
                                                  (uint32_t)v4[2] | ((uint32_t)v4[3] << 16));
    } else {
      const size_t row = (size_t)share * a.rows + blockIdx.x / kHkv * (2 * kCt) + token;
      const size_t pt = row * kHq + head;
      *(f32x4*)(a.part_o + pt * kD + d) = ot;
      if (d == 0) *(float2*)(a.part_ml + pt * 2) = make_float2(mt, lt);
    }
  }
}

// Long chunks: a workgroup takes kTokens tokens x the 8 heads of a kv head (columns
// (token, head)) through the sequence's keys in blocks of 64, a wave 4 tokens: one
// column tile of 32.  Bound by the vector ALUs (per 32 x 32 scores 16 exponentials,
// 16 multiply-adds, 8 conversions and 8 dot products of a wave against 8 matrix
// products), so:
//  * v_mfma_f32_32x32x16_bf16: S^T = K Q^T leaves lane (column l % 32, half h =
//    l / 32) the keys 8 (i / 4) + 4 h + i % 4 of a 32-key tile in elements i = 0 ..
//    15, which are, packed to bf16, the operands of two products O^T += V^T P^T over 16
//    keys each.  V^T's tile keeps its 4-key quads in that order: lane half h of
//    product m reads quads 4 m + h and 4 m + 2 + h as one 16-byte unit.
//  * p enters as one bf16 rounding, and the sum takes the rounded p (v_dot2): a
//    weight is off by at most half a bf16 step, as the output's own rounding is,
//    and where few keys matter the two cancel.  (The cached values' own half step is
//    sixteen times as large.)  Errors against 64 bits are 0.0020 to 0.0021; in two
//    pieces, as decode has p, 0.0017, for half as many products again and 40 more
//    vector instructions a tile: 4096 tokens 223 us instead of 151, 300 over 6000 72
//    instead of 55.
//  * No row maximum: the softmax's reference point m is the maximum of the
//    first keys a column sees, and stays.  Larger scores only make p larger than
//    1, which fp32 and bf16 carry; a wave takes new maxima, rescales and computes its
//    p anew only when some column's sum over a tile passes 2^24 (or m is not set:
//    -m = inf gives an infinite or NaN sum).
//  * 128 registers (the form in halves spills one), so that four waves share a SIMD: a
//    wave alone issues a vector instruction every 8 cycles, and one's matrix products can
//    run under the others' exponentials.  They do so little: at 4096 tokens the matrix
//    cores are busy 36% of the time and the vector units 55%.  (64 columns a wave,
//    two waves, with the products of one tile and the exponentials of the next
//    interleaved by hand: the same time.)
// The next block's codes are loaded to registers during a block's products, then
// converted once for all waves, k with its scale, v with its keys', into LDS (bf16,
// rows of 128 bytes whose 16-byte units are XORed with the row's bits 1 .. 3, so
// 16 rows of one unit spread over all banks); one barrier per block.
// A row that must not be used (255) is NaN in k and 0 in v.
//
// 64 tokens halve the conversions per column, but a CU holds one workgroup and not
// two, the last ones leave more of the chip idle, and a window's edges are masked in
// more columns: 4096 tokens 157 us against 161, 2048 tokens 72 against 54, 4096 with
// window 128 44 against 33.  So they are taken without a window where they are two
// rounds or more of the chip.  With kHalves = 2 the workgroup's second half takes the
// other blocks of its share, and the states meet in LDS.  At 4096 tokens 865 to 905
// TFLOP/s (a library product of 8192^3 reaches 1314), 300 over 6000 530 with the merge.
constexpr int kTileBytes = kFp8Block * kD * 2;
constexpr int tile_threads(int tokens, int halves) { return 16 * tokens * halves; }
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// max over lanes l and l ^ 32
__device__ __forceinline__ float half_max(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

template <int kTokens, bool kSplit, int kHalves>
__global__ __launch_bounds__(tile_threads(kTokens, kHalves))
__attribute__((amdgpu_waves_per_eu(4))) void fp8_tile_kernel(RowsArgs a) {
  constexpr int kWaves = kTokens / 4;  // of a half
  __shared__ __align__(16) uint8_t lds[kHalves][2][2][kTileBytes];
  // x: (tile from the last, which sees the most keys; sequence; kv head), y: split
  const int hk = blockIdx.x % kHkv, total = gridDim.x / kHkv, batch = total / a.tiles;
  int rest = blockIdx.x / kHkv;
  // An XCD's 32 CUs take the second 32 workgroups beside the first: in reverse, so that
  // the longest has the shortest beside it (2048 tokens 59 -> 54 us)
  if (kTokens == 32 && rest >= 32 && rest < 64) rest = min(total, 64) - 1 - (rest - 32);
  const int b = rest % batch, tile = a.tiles - 1 - rest / batch;
  const int qb = a.q_indptr[b], qn = a.q_indptr[b + 1] - qb, t0 = tile * kTokens;
  if (t0 >= qn) return;
  const int nt = min(kTokens, qn - t0), row0 = qb + t0;
  const int L = a.kv_len[b], pos = L - qn + t0;
  const Sight sight(pos, nt, a.window);
  const Shares shares(sight.blocks, kSplit ? a.splits : 1, a.least);
  const int share = kSplit ? blockIdx.y : 0;
  if (share >= max(shares.used, 1)) return;
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6) % kWaves;
  const int half = kHalves == 1 ? 0 : __builtin_amdgcn_readfirstlane(t >> 6) / kWaves;
  const int c = lane & 31, h = lane >> 5;
  const PageList pages{a.page_indices + a.page_indptr[b],
                       a.page_indptr[b + 1] - a.page_indptr[b], a.num_pages};
  const int last_page = max(0, min(pages.count - 1, (L - 1) / kPage));
  const int begin0 = sight.first + share * shares.each;
  const int end0 = min(begin0 + shares.each, sight.first + sight.blocks);
  const int most = (end0 - begin0 + kHalves - 1) / kHalves;  // blocks of a half
  const int begin = begin0 + half * most, end = min(begin + most, end0);
  uint8_t(*const kt)[kTileBytes] = lds[half][0];
  uint8_t(*const vt)[kTileBytes] = lds[half][1];

  // Staging: waves 0 .. 3 take k, waves 4 .. 7 v of page `wave & 3` of a block: lane
  // the 16 dims 16 (l % 4) .. of key l / 4, or the four keys of quad l / 16 in v's unit
  // l % 16; both take their keys' scales.
  const int mine = wave & 3, quad = 4 * mine + (lane >> 4);
  const bool is_v = wave & 4, stages = kWaves == 8 || wave < 8;
  const unsigned part = (is_v ? kFp8V : 0) + hk * kFp8Head + lane * 16;
  const unsigned spart = kFp8Scales + hk * 2 * kPage + (lane >> 4) * 4;
  struct Raw {
    u32x4 codes;
    uint32_t ks, vs;
  };
  // the pages of 64 blocks at a time, one a lane (past the last block: its last page again)
  int ids = 0;
  auto fetch_ids = [&](int blk) {
    ids = pages.count > 0 ? pages.clamp(pages.ids[min(4 * (blk + lane) + mine, last_page)]) : 0;
  };
  auto load = [&](Raw& x, int blk) {
    const int i = (blk - begin) & 63;
    if (i == 0 && blk > begin) fetch_ids(blk);
    const uint8_t* page = a.cache + (size_t)(unsigned)__builtin_amdgcn_readlane(ids, i) * kFp8Page;
    x.codes = *(const u32x4*)(page + part);
    x.ks = *(const uint32_t*)(page + spart);
    x.vs = *(const uint32_t*)(page + spart + kPage);
  };
  auto store = [&](Raw& x, int buf, int kb) {
    if (!is_v) {
      const int byte = 8 * ((lane >> 2) & 3), key = 16 * mine + (lane >> 2);
      const uint32_t sk = (x.ks >> byte) & 255u, sv = (x.vs >> byte) & 255u;
      const bool bad = max(sk, sv) == kFp8BadScale;
      const float scale = __uint_as_float(min(sk, kFp8BadScale - 1u) << 23);
#pragma unroll
      for (int j = 0; j < 4; ++j) x.codes[j] = bad ? kFp8NanCodes : x.codes[j];
      uint8_t* row = kt[buf] + key * 128;
      const int swz = (key >> 1) & 7, u = 2 * (lane & 3);
      *(bf16x8*)(row + ((u ^ swz) << 4)) = fp8_to_bf16(x.codes[0], x.codes[1], scale);
      *(bf16x8*)(row + (((u + 1) ^ swz) << 4)) = fp8_to_bf16(x.codes[2], x.codes[3], scale);
      return;
    }
    const int n = quad & 7, r = lane & 15;
    const int unit = 4 * (quad >> 3) + 2 * (n >> 2) + (n & 1), half = (n >> 1) & 1;
    uint32_t keep = ~0u;
    if (kb + kFp8Block > L) {  // stale codes past the sequence's end may be NaN
      const int m = min(max(L - (kb + 4 * quad), 0), 4);
      keep = m == 4 ? ~0u : (1u << (8 * m)) - 1u;
    }
    float s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      s[j] = __uint_as_float(min((x.vs >> (8 * j)) & 255u, kFp8BadScale - 1u) << 23);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      const uint32_t w = x.codes[dt] & keep;
      auto pair = [&](float s0, float s1, auto hi) {  // two keys, each with its scale
        const auto x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s0, decltype(hi)::value);
        const auto x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s1, decltype(hi)::value);
        return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, x1),
                                     __builtin_bit_cast(uint32_t, x0), 0x07060100u);
      };
      const uint32_t p0 = pair(s[0], s[1], std::false_type{});
      const uint32_t p1 = pair(s[2], s[3], std::true_type{});
      const int d = 16 * dt + r;
      *(uint2*)(vt[buf] + d * 128 + ((unit ^ ((d >> 1) & 7)) << 4) + 8 * half) = make_uint2(p0, p1);
    }
  };

  // the first blocks' codes and q are on their way at once
  Raw raw, raw0;
  if (stages && begin < end) {
    fetch_ids(begin);
    load(raw0, begin);
    load(raw, begin + 1);
  }
  const int token = min(4 * wave + (c >> 3), nt - 1);
  const uint16_t sink = a.sinks[hk * kGroup + (c & 7)];
  bf16x8 qv[4];
  {
    const u32x4* src =
        (const u32x4*)(a.q + ((size_t)(row0 + token) * kHq + hk * kGroup + (c & 7)) * kD);
#pragma unroll
    for (int s = 0; s < 4; ++s) qv[s] = moe::as_bf16x8(src[2 * s + h]);
  }
  const int qpos = pos + token - 4 * h;  // element i's key is 8 (i / 4) + i % 4 from 4 h on
  const unsigned reach = a.window > 0 ? a.window : 0x7FFFFFFFu;  // keys back that a token sees
  const moe::bf16x2 ones = {(__bf16)1.0f, (__bf16)1.0f};
  f32x16 o[2];
  float mneg = INFINITY, l = 0.f;
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;

  if (stages && begin < end) store(raw0, 0, begin * kFp8Block);
  moe::lds_barrier();
  int buf = 0;
  auto run = [&](auto masked, int from, int to) __attribute__((always_inline)) {
    for (int blk = from; blk < to; ++blk) {
      const int kb = blk * kFp8Block;
#pragma unroll
      for (int kt32 = 0; kt32 < 2; ++kt32) {
        f32x16 s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          const bf16x8 ka = *(const bf16x8*)(kt[buf] + (32 * kt32 + c) * 128 +
                                             (((2 * st + h) ^ ((c >> 1) & 7)) << 4));
          s = mfma32(ka, qv[st], s);
        }
        if constexpr (decltype(masked)::value) {
          const int back = qpos - kb - 32 * kt32;  // of the first element's key behind the token
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[i] = (unsigned)(back - 8 * (i >> 2) - (i & 3)) < reach ? s[i] : -INFINITY;
        }
        moe::bf16x2 p[8];
        float ps;
        auto exps = [&](float mn) __attribute__((always_inline)) {
          ps = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            p[i][0] = (__bf16)__builtin_amdgcn_exp2f(fmaf(s[2 * i], a.c2, mn));
            p[i][1] = (__bf16)__builtin_amdgcn_exp2f(fmaf(s[2 * i + 1], a.c2, mn));
            ps = __builtin_amdgcn_fdot2_f32_bf16(p[i], ones, ps, false);
          }
        };
        exps(mneg);
        if (__any(!(ps < kFp8Most))) {
          float mx = s[0];
#pragma unroll
          for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
          const float m = -mneg, mn = fmaxf(m, half_max(mx) * a.c2);
          const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
          for (int dt = 0; dt < 2; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
          l *= alpha;
          mneg = -mn;
          exps(mn == -INFINITY ? 0.0f : -mn);
        }
        l += ps;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          bf16x8 pb;
#pragma unroll
          for (int j = 0; j < 8; ++j) pb[j] = p[4 * m + (j >> 1)][j & 1];
#pragma unroll
          for (int dt = 0; dt < 2; ++dt) {
            const bf16x8 va = *(const bf16x8*)(vt[buf] + (32 * dt + c) * 128 +
                                               (((4 * kt32 + 2 * m + h) ^ ((c >> 1) & 7)) << 4));
            o[dt] = mfma32(va, pb, o[dt]);
          }
        }
      }
      if (stages && blk + 1 < end) store(raw, buf ^ 1, kb + kFp8Block);
      if (stages && blk + 2 < end) load(raw, blk + 2);  // in flight during the next's products
      moe::lds_barrier();
      buf ^= 1;
    }
  };
  // blocks that every token sees whole: from whole0 to whole1
  const int whole1 = max(begin, min(end, (pos + 1) / kFp8Block));
  const int seen0 = (sight.last - a.window) / kFp8Block + 1;
  const int whole0 = min(whole1, a.window <= 0 ? begin : max(begin, seen0));
  run(std::true_type{}, begin, whole0);
  run(std::false_type{}, whole0, whole1);
  run(std::true_type{}, whole1, end);

  float lt = l + __shfl_xor(l, 32, kWave);
  if constexpr (kHalves == 2) {
    // the second half's states into the first's, through the tiles' LDS
    __shared__ float2 ml[kWaves][32];
    for (int i = max(end - begin, 0); i < most; ++i) moe::lds_barrier();
    f32x4* const part = (f32x4*)&lds[0][0][0][0] + wave * 8 * kWave + lane;
    if (half == 1) {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        part[q * kWave] = f32x4{o[q >> 2][4 * (q & 3)], o[q >> 2][4 * (q & 3) + 1],
                                o[q >> 2][4 * (q & 3) + 2], o[q >> 2][4 * (q & 3) + 3]};
      if (h == 0) ml[wave][c] = make_float2(-mneg, lt);
    }
    moe::lds_barrier();
    if (half == 1) return;
    const float2 other = ml[wave][c];
    const float m = fmaxf(-mneg, other.x);
    const float w0 = -mneg == -INFINITY && lt == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(-mneg - m);
    const float w1 =
        other.x == -INFINITY && other.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(other.x - m);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const f32x4 po = part[q * kWave];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[q >> 2][4 * (q & 3) + j] = fmaf(po[j], w1, o[q >> 2][4 * (q & 3) + j] * w0);
    }
    lt = fmaf(other.y, w1, lt * w0);
    mneg = -m;
  }
  const bool alone = shares.used <= 1;
  if (4 * wave + (c >> 3) >= nt) return;
  const size_t at = (size_t)(row0 + token) * kHq + hk * kGroup + (c & 7);
  if (alone) {
    const float f = sink_share(lt, -mneg, sink);
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        uint16_t v4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v4[j] = f2bf(o[dt][i + j] * f);
        *(uint2*)(a.out + at * kD + 32 * dt + 2 * i + 4 * h) =
            make_uint2((uint32_t)v4[0] | ((uint32_t)v4[1] << 16),
                       (uint32_t)v4[2] | ((uint32_t)v4[3] << 16));
      }
  } else {
    const size_t pt = ((size_t)share * a.rows + (b * a.tiles + tile) * kTokens + token) * kHq +
                      hk * kGroup + (c & 7);
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *(f32x4*)(a.part_o + pt * kD + 32 * dt + 2 * i + 4 * h) =
            f32x4{o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]};
    if (h == 0) *(float2*)(a.part_ml + pt * 2) = make_float2(-mneg, lt);
  }
}

// The splits of a chunk's tiles merged: one wave four rows (token, head), a thread
// four dimensions, eight splits' loads in flight.  `tokens`: of a tile.
__global__ __launch_bounds__(256) void fp8_merge_kernel(RowsArgs a, int tokens) {
  const int b = blockIdx.x / a.tiles, t0 = blockIdx.x % a.tiles * tokens;
  const int qb = a.q_indptr[b], qn = a.q_indptr[b + 1] - qb;
  const int i = blockIdx.y * 16 + (threadIdx.x >> 4);  // (token of the tile, head)
  const int token = i / kHq, head = i % kHq, d = (threadIdx.x & 15) * 4;
  if (token >= tokens || t0 + token >= qn) return;
  const Sight sight(a.kv_len[b] - qn + t0, min(tokens, qn - t0), a.window);
  const int used = Shares(sight.blocks, a.splits, a.least).used;
  if (used <= 1) return;  // written already
  const size_t at = ((size_t)blockIdx.x * tokens + token) * kHq + head;
  const size_t step = (size_t)a.rows * kHq;
  float m = -INFINITY, l = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < used; s0 += 8) {
    float2 ml[8];
    f32x4 po[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const size_t pt = at + (size_t)min(s0 + j, used - 1) * step;
      ml[j] = *(const float2*)(a.part_ml + pt * 2);
      po[j] = *(const f32x4*)(a.part_o + pt * kD + d);
    }
    float mn = m;
#pragma unroll
    for (int j = 0; j < 8; ++j) mn = s0 + j < used ? fmaxf(mn, ml[j].x) : mn;
    const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    if (s0 > 0) {
      l *= alpha;
#pragma unroll
      for (int q = 0; q < 4; ++q) o[q] *= alpha;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (s0 + j >= used) continue;
      const float w = ml[j].x == -INFINITY && ml[j].y == 0.0f
                          ? 0.0f : __builtin_amdgcn_exp2f(ml[j].x - mn);
      l = fmaf(ml[j].y, w, l);
#pragma unroll
      for (int q = 0; q < 4; ++q) o[q] = fmaf(po[j][q], w, o[q]);
    }
    m = mn;
  }
  const float f = sink_share(l, m, a.sinks[head]);
  uint16_t v4[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) v4[q] = f2bf(o[q] * f);
  *(uint2*)(a.out + ((size_t)(qb + t0 + token) * kHq + head) * kD + d) =
      make_uint2((uint32_t)v4[0] | ((uint32_t)v4[1] << 16),
                 (uint32_t)v4[2] | ((uint32_t)v4[3] << 16));
}

}  // namespace attn

// ---------------------------------------------------------------------------
// Launchers (argument checks live in the C ABI, attn_capi.hip)
extern "C" {

int attn_launch_fp8_quantize(const void* src, int src_pages, const int* src_slots, int n,
                             void* cache, int num_pages, const int* slots, hipStream_t s) {
  hipLaunchKernelGGL(attn::fp8_quantize_kernel, dim3((n - 1) / 16 + 1), dim3(256), 0, s,
                     (const uint8_t*)src, src_pages, src_slots, n, (uint8_t*)cache, num_pages,
                     slots);
  return hipGetLastError() == hipSuccess ? 0 : -6;
}

int attn_launch_fp8_read(const void* cache, int num_pages, const int* slots, int n, void* k_out,
                         void* v_out, hipStream_t s) {
  hipLaunchKernelGGL(attn::fp8_read_kernel, dim3((n - 1) / 16 + 1), dim3(256), 0, s,
                     (const uint8_t*)cache, num_pages, slots, n, (uint16_t*)k_out,
                     (uint16_t*)v_out);
  return hipGetLastError() == hipSuccess ? 0 : -6;
}

// part_o [splits][batch][64][64], part_ml [splits][batch][64][2], splits <= 64
int attn_launch_fp8_decode(const void* q, int batch, const void* cache, const int* page_indptr,
                           const int* page_indices, int num_pages, const int* kv_len,
                           int64_t max_span, int window, float sm_scale, const void* sinks,
                           int splits, int least, float* part_o, float* part_ml, int* arrive,
                           void* out, hipStream_t s) {
  if (splits < 1 || splits > 64) return -6;
  const attn::RowsArgs a{(const uint16_t*)q, nullptr, (const uint8_t*)cache, page_indptr,
                         page_indices, kv_len, (const uint16_t*)sinks, (uint16_t*)out, part_o,
                         part_ml, arrive, max_span, num_pages, window, splits, least, batch, 1,
                         sm_scale * attn::kLog2e};
  hipLaunchKernelGGL(attn::fp8_decode_kernel, dim3(attn::kHkv * batch, splits), dim3(256),
                     0, s, a);
  return hipGetLastError() == hipSuccess ? 0 : -6;
}

// tokens: of a tile, 2, 4, 32 or (not split) 64; part_o [splits][rows][64][64], part_ml
// [splits][rows][64][2] where splits > 1.  A launch holds less than 2^32 threads: more
// tiles go in launches of some sequences each, which are never split ones (their
// workgroups fit the chip at once).
int attn_launch_fp8_chunk(const void* q, const int* q_indptr, int batch, int max_q_len,
                          const void* cache, const int* page_indptr, const int* page_indices,
                          int num_pages, const int* kv_len, int window, float sm_scale,
                          const void* sinks, void* out, int tokens, int splits, int halves,
                          int rows, float* part_o, float* part_ml, hipStream_t s) {
  if (tokens == 64 ? splits != 1 || halves != 1 : tokens != 32 && halves != 1) return -6;
  const int tiles = (max_q_len + tokens - 1) / tokens;
  const int threads = tokens >= 32 ? attn::tile_threads(tokens, halves) : 256;
  const int64_t room = (((int64_t)1 << 32) - 1) / ((int64_t)threads * attn::kHkv * tiles);
  if (room < 1 || (splits > 1 && batch > room)) return -6;
  for (int b = 0, most = (int)(room < batch ? room : batch); b < batch; b += most) {
    const int group = batch - b < most ? batch - b : most;
    const attn::RowsArgs a{(const uint16_t*)q, q_indptr + b, (const uint8_t*)cache,
                           page_indptr + b, page_indices, kv_len + b, (const uint16_t*)sinks,
                           (uint16_t*)out, part_o, part_ml, nullptr, 0, num_pages, window, splits,
                           4 * halves, rows, tiles, sm_scale * attn::kLog2e};
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(attn::kHkv * group * tiles, splits), dim3(threads), 0, s, a);
    };
    if (tokens == 2)
      go(attn::fp8_rows_kernel<1>);
    else if (tokens == 4)
      go(attn::fp8_rows_kernel<2>);
    else if (tokens == 64)
      go(attn::fp8_tile_kernel<64, false, 1>);
    else if (halves == 2)
      go(attn::fp8_tile_kernel<32, true, 2>);
    else if (splits > 1)
      go(attn::fp8_tile_kernel<32, true, 1>);
    else
      go(attn::fp8_tile_kernel<32, false, 1>);
    if (hipGetLastError() != hipSuccess) return -6;
    if (splits > 1) {
      hipLaunchKernelGGL(attn::fp8_merge_kernel, dim3(group * tiles, tokens * attn::kHq / 16),
                         dim3(256), 0, s, a, tokens);
      if (hipGetLastError() != hipSuccess) return -6;
    }
  }
  return 0;
}

}  // extern "C"
