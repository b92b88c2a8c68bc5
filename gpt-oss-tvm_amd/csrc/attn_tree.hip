// Attention of trees of drafted tokens over the paged cache (gfx950), bf16 and 8-bit.
//
// A sequence of c cached tokens holds its tree's node i at index c + i of its pages; node i sees
// the cached keys (those of the window, where there is one) and the nodes that its mask has:
//   out = sum_j p_j v_j / (sum_j p_j + exp(sink)),  p_j = exp(sm_scale q . k_j)
// rounded to bf16 once; a node that sees no key gets 0.
#include "attn_common.h"

namespace attn {

constexpr int kHeadBytes = kPage * kD * 2;           // of a bf16 page's k or v of one head
constexpr int kBfPage = 2 * kHkv * kHeadBytes;
constexpr float kTreeLog2e = 1.4426950408889634f;

struct TreeArgs {
  const uint16_t* q;
  const int* q_indptr;
  const uint32_t* mask;  // [rows][words]
  const int* positions;
  const uint8_t* cache;
  const int* page_indptr;
  const int* page_indices;
  const int* kv_len;
  const uint16_t* sinks;
  uint16_t* out;
  int words, num_pages, window;
  float c2;  // sm_scale log2(e)
};

// One token and kv head a workgroup, 32 threads a head: a thread a key of 32 for the scores,
// two dimensions for the output.
template <bool kFp8>
__global__ __launch_bounds__(256) void tree_kernel(TreeArgs a) {
  const int b = blockIdx.y, node = blockIdx.x / kHkv, hk = blockIdx.x % kHkv;
  const int qb = a.q_indptr[b], qn = a.q_indptr[b + 1] - qb;
  if (node >= qn) return;
  const int row = qb + node, L = a.kv_len[b], cached = L - qn;
  const int t = threadIdx.x, h = t >> 5, i = t & 31, head = hk * kGroup + h;
  const PageList pages{a.page_indices + a.page_indptr[b],
                       a.page_indptr[b + 1] - a.page_indptr[b], a.num_pages};
  const int pos = max(a.positions[row], cached);
  const int lo = a.window > 0 ? pos - a.window + 1 : 0;  // the first position that is seen
  const uint16_t* const q = a.q + ((size_t)row * kHq + head) * kD;
  auto seen = [&](int key) {
    if (key < 0 || key >= L || pages.count <= 0) return false;
    if (key < cached) return key >= lo;
    const int j = key - cached;
    return (a.mask[(size_t)row * a.words + (j >> 5)] >> (j & 31) & 1) != 0 &&
           max(a.positions[qb + j], cached) >= lo;
  };
  auto value = [&](const uint8_t* page, int kv, int slot, int d) {
    if constexpr (kFp8) {
      const uint32_t s = page[fp8_scale_at(hk, kv, slot)];
      const uint8_t code =
          kv ? page[fp8_v_at(hk, slot, d)] : page[hk * kFp8Head + slot * kFp8Row + d];
      return s == kFp8BadScale ? NAN : moe::e4m3_byte<0>(code) * __uint_as_float(s << 23);
    } else {
      return bf2f(((const uint16_t*)(page + (kv * kHkv + hk) * kHeadBytes))[slot * kD + d]);
    }
  };
  auto page_at = [&](int key) {
    return a.cache + (size_t)pages.page_of(key) * (kFp8 ? kFp8Page : kBfPage);
  };
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int k0 = max(min(lo, cached), 0) & ~31; k0 < L; k0 += 32) {
    const int key = k0 + i;
    float s = -INFINITY;
    if (seen(key)) {
      const uint8_t* page = page_at(key);
      s = 0.f;
      for (int d = 0; d < kD; ++d) s = fmaf(bf2f(q[d]), value(page, 0, key % kPage, d), s);
      s *= a.c2;
    }
    float mx = s;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, kWave));
    const float mn = fmaxf(m, mx);
    const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    const float p = s == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s - mn);
    m = mn;
    l = l * alpha + p;
    o0 *= alpha;
    o1 *= alpha;
    for (int j = 0; j < 32; ++j) {
      const float pj = __shfl(p, (t & 32) + j, kWave);
      if (!seen(k0 + j)) continue;
      const uint8_t* page = page_at(k0 + j);
      o0 = fmaf(pj, value(page, 1, (k0 + j) % kPage, 2 * i), o0);
      o1 = fmaf(pj, value(page, 1, (k0 + j) % kPage, 2 * i + 1), o1);
    }
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) l += __shfl_xor(l, off, kWave);
  const float f =
      l == 0.0f ? 0.0f
                : 1.0f / (l + __builtin_amdgcn_exp2f(fmaf(bf2f(a.sinks[head]), kTreeLog2e, -m)));
  *(uint32_t*)(a.out + ((size_t)row * kHq + head) * kD + 2 * i) =
      (uint32_t)f2bf(o0 * f) | ((uint32_t)f2bf(o1 * f) << 16);
}

}  // namespace attn

extern "C" {

int attn_launch_tree(const void* q, const int* q_indptr, int batch, int max_q_len,
                     const void* mask, int words, const int* positions, const void* cache,
                     bool fp8, const int* page_indptr, const int* page_indices, int num_pages,
                     const int* kv_len, int window, float sm_scale, const void* sinks, void* out,
                     hipStream_t s) {
  const attn::TreeArgs a{(const uint16_t*)q, q_indptr, (const uint32_t*)mask, positions,
                         (const uint8_t*)cache, page_indptr, page_indices, kv_len,
                         (const uint16_t*)sinks, (uint16_t*)out, words, num_pages, window,
                         sm_scale * attn::kTreeLog2e};
  const dim3 grid(attn::kHkv * max_q_len, batch);
  if (fp8)
    hipLaunchKernelGGL(attn::tree_kernel<true>, grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(attn::tree_kernel<false>, grid, dim3(256), 0, s, a);
  return hipGetLastError() == hipSuccess ? 0 : -6;
}

}  // extern "C"
