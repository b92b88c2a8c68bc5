// Rows and pages of the KV cache moved in all layers at once (gfx950): the nodes of a drafted
// tree that the model accepted, behind the cached tokens; the pages of a sequence that another
// one goes on from.
#include "attn_common.h"

namespace attn {

constexpr int kMoveBfHead = kPage * kD * 2;
constexpr int kMoveBfPage = 2 * kHkv * kMoveBfHead;
constexpr int kMoveNodes = 1024;  // of a tree at most

struct CommitArgs {
  uint8_t* cache;  // [layers][num_pages] pages
  const int* page_indptr;
  const int* page_indices;
  const int* kv_len;
  const int* q_indptr;
  const int* tokens;
  const int* parents;
  const int* chosen;
  int* path;   // [rows]
  int* count;  // [batch]
  int* next;   // [batch]
  int batch, rows, num_pages, max_q;
};

// The walk, by one wave: at most kMoveNodes nodes, each step to a later node, so it ends.
// Leaves the path in LDS and returns its length.
__device__ __forceinline__ int tree_walk(const CommitArgs& a, int qb, int qn, int* path) {
  const int lane = threadIdx.x;
  int at = 0, n = 0;
  while (true) {
    if (lane == 0) path[n] = at;
    ++n;
    const int want = a.chosen[qb + at];
    int child = qn;
    for (int j0 = at + 1; j0 < qn && child == qn; j0 += kWave) {
      const int j = j0 + lane;
      const bool hit = j < qn && a.parents[qb + j] == at && a.tokens[qb + j] == want;
      const uint64_t who = __ballot(hit);
      if (who) child = j0 + __builtin_ctzll(who);
    }
    if (child == qn) return n;
    at = child;
  }
}

// Grid (layers, batch): a workgroup walks its sequence's tree (all of them the same path) and
// moves its layer's rows, a row at a time: the path's nodes ascend and none comes before its
// place, so no row is overwritten before it is read.
template <bool kFp8>
__global__ __launch_bounds__(256) void tree_commit_kernel(CommitArgs a) {
  __shared__ int path[kMoveNodes];
  __shared__ int length;
  const int layer = blockIdx.x, b = blockIdx.y, t = threadIdx.x;
  const int qb = a.q_indptr[b], qn = min(a.q_indptr[b + 1] - qb, a.max_q);
  if (t < kWave) {
    const int n = qn > 0 ? tree_walk(a, qb, qn, path) : 0;
    if (t == 0) length = n;
  }
  __syncthreads();
  const int n = length;
  if (layer == 0) {
    for (int i = t; i < qn; i += 256) a.path[qb + i] = i < n ? path[i] : -1;
    if (t == 0) {
      a.count[b] = n;
      a.next[b] = n > 0 ? a.chosen[qb + path[n - 1]] : -1;
    }
    if (b == a.batch - 1)
      for (int i = a.q_indptr[a.batch] + t; i < a.rows; i += 256) a.path[i] = -1;
  }
  const int cached = a.kv_len[b] - (a.q_indptr[b + 1] - qb);
  const PageList pages{a.page_indices + a.page_indptr[b],
                       a.page_indptr[b + 1] - a.page_indptr[b], a.num_pages};
  constexpr int kBytes = kFp8 ? kFp8Page : kMoveBfPage;
  uint8_t* const data = a.cache + (size_t)layer * a.num_pages * kBytes;
  for (int i = 0; i < n; ++i) {
    const int from = cached + path[i], to = cached + i;
    if (from == to || from < 0 || to < 0 || pages.count <= 0) continue;
    const uint8_t* src = data + (size_t)pages.page_of(from) * kBytes;
    uint8_t* dst = data + (size_t)pages.page_of(to) * kBytes;
    const int fs = from % kPage, ts = to % kPage;
    if constexpr (kFp8) {
      if (t < 32) {  // (head, 16 bytes of k)
        const int h = t >> 2, u = (t & 3) * 16;
        *(u32x4*)(dst + h * kFp8Head + ts * kFp8Row + u) =
            *(const u32x4*)(src + h * kFp8Head + fs * kFp8Row + u);
      } else if (t >= 64 && t < 80) {
        const int h = (t - 64) >> 1, kv = t & 1;
        dst[fp8_scale_at(h, kv, ts)] = src[fp8_scale_at(h, kv, fs)];
      }
      for (int j = t; j < kHkv * kD; j += 256)
        dst[fp8_v_at(j / kD, ts, j % kD)] = src[fp8_v_at(j / kD, fs, j % kD)];
    } else if (t < 128) {
      const int h = t >> 3, u = (t & 7) * 16;
      *(u32x4*)(dst + h * kMoveBfHead + ts * (kD * 2) + u) =
          *(const u32x4*)(src + h * kMoveBfHead + fs * (kD * 2) + u);
    }
    __syncthreads();
  }
}

// Pages copied in every layer: grid (pages, layers).
__global__ __launch_bounds__(256) void copy_pages_kernel(uint8_t* __restrict__ cache,
                                                         int num_pages, int units,
                                                         const int* __restrict__ src,
                                                         const int* __restrict__ dst) {
  const int from = src[blockIdx.x], to = dst[blockIdx.x];
  if ((unsigned)from >= (unsigned)num_pages || (unsigned)to >= (unsigned)num_pages) return;
  u32x4* const data = (u32x4*)cache + (size_t)blockIdx.y * num_pages * units;
  for (int i = threadIdx.x; i < units; i += 256)
    data[(size_t)to * units + i] = data[(size_t)from * units + i];
}

}  // namespace attn

extern "C" {

int attn_launch_tree_commit(void* cache, int layers, int num_pages, bool fp8,
                            const int* page_indptr, const int* page_indices, const int* kv_len,
                            const int* q_indptr, int batch, int rows, int max_q_len,
                            const int* tokens, const int* parents, const int* chosen, int* path,
                            int* count, int* next, hipStream_t s) {
  const attn::CommitArgs a{(uint8_t*)cache, page_indptr, page_indices, kv_len, q_indptr, tokens,
                           parents, chosen, path, count, next, batch, rows, num_pages, max_q_len};
  const dim3 grid(layers, batch);
  if (fp8)
    hipLaunchKernelGGL(attn::tree_commit_kernel<true>, grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(attn::tree_commit_kernel<false>, grid, dim3(256), 0, s, a);
  return hipGetLastError() == hipSuccess ? 0 : -6;
}

int attn_launch_copy_pages(void* cache, int layers, int num_pages, int page_bytes, const int* src,
                           const int* dst, int n, hipStream_t s) {
  hipLaunchKernelGGL(attn::copy_pages_kernel, dim3(n, layers), dim3(256), 0, s, (uint8_t*)cache,
                     num_pages, page_bytes / 16, src, dst);
  return hipGetLastError() == hipSuccess ? 0 : -6;
}

}  // extern "C"
