// Rows and pages of the KV cache moved in all layers at once (gfx950): the nodes of a drafted
// tree that the model accepted, behind the cached tokens; the pages of a sequence that another
// one goes on from.
#include <stdint.h>

#include <algorithm>

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
  int batch, rows, num_pages;
  int room;  // the trees' most nodes, at most kMoveNodes
};

// The walk from node 0 along the chosen tokens, by one wave: at most kMoveNodes nodes, each step to
// a later one, so it ends.  A tree of up to 64 nodes lies in the wave's registers, a lane a node; a
// larger one in LDS.  Leaves the path in LDS and returns its length, the number of its nodes that
// are in their places and the last token chosen.
struct Walk {
  int length, still, last;
};
__device__ __forceinline__ Walk tree_walk(const CommitArgs& a, int qb, int qn, int* path,
                                          int* parents, int* tokens, int* chosen) {
  const int lane = threadIdx.x & 63;
  int at = 0, n = 0, still = 0, want = -1;
  if (qn <= kWave) {
    const int j = qb + min(lane, qn - 1);
    const int parent = a.parents[j], token = a.tokens[j], choice = a.chosen[j];
    while (true) {
      if (lane == 0) path[n] = at;
      still += at == n;
      ++n;
      want = __builtin_amdgcn_readlane(choice, at);
      const uint64_t who =
          __ballot(lane > at && lane < qn && parent == at && token == want);
      if (who == 0) return Walk{n, still, want};
      at = __builtin_ctzll(who);
    }
  }
  for (int j = lane; j < qn; j += kWave) {
    parents[j] = a.parents[qb + j];
    tokens[j] = a.tokens[qb + j];
    chosen[j] = a.chosen[qb + j];
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (one wave wrote them and reads them)
  while (true) {
    if (lane == 0) path[n] = at;
    still += at == n;
    ++n;
    want = chosen[at];
    int child = qn;
    for (int j0 = at + 1; j0 < qn && child == qn; j0 += kWave) {
      const int j = min(j0 + lane, qn - 1);
      const uint64_t who =
          __ballot(j0 + lane < qn && parents[j] == at && tokens[j] == want);
      if (who) child = j0 + __builtin_ctzll(who);
    }
    if (child == qn) return Walk{n, still, want};
    at = child;
  }
}

// Grid (layers, batch): a workgroup walks its sequence's tree (all of them the same way: cheaper
// than a launch of its own) and moves its layer's rows, a lot of at most four at a time, all read
// before the first is written.  The path's nodes ascend and none comes before its place, so no row
// is overwritten by an earlier lot before it is read.  A lot ends where the destination's index is a
// multiple of four: v's codes lie four tokens to a word, and a lot's are put into their words in
// registers and written with what else those words hold.
// Bound by the loads that wait for one another (tables, nodes, page ids, rows) and, where there is
// more to move, by lines that are touched in part: 64 trees of 26 nodes in 36 layers of an 8-bit
// cache 8.7 us, 4 of them up to the page ids, for 17 MB of lines (3.5 us at a copy's rate).  v's
// codes written a byte at a time, lots of four rows 9.8, of eight 11.1; a row at a time with a
// barrier each and the walk's steps from memory 13.3; two layers a workgroup, one after the other,
// 13.4.  One tree of 8 nodes in 24 layers of a bf16 cache 2.2 us.
constexpr int kMoveRows = 4;

template <bool kFp8>
__global__ __launch_bounds__(256) void tree_commit_kernel(CommitArgs a) {
  extern __shared__ int move_lds[];  // path, sources' and destinations' slots, larger trees' nodes
  __shared__ Walk walk;
  int *const path = move_lds, *const source = path + a.room, *const dest = source + a.room;
  const int b = blockIdx.y, t = threadIdx.x;
  const int qb = a.q_indptr[b], nodes_in = a.q_indptr[b + 1] - qb;
  const int qn = min(min(nodes_in, a.room), a.rows - qb);
  const int cached = a.kv_len[b] - nodes_in;
  const PageList pages{a.page_indices + a.page_indptr[b],
                       a.page_indptr[b + 1] - a.page_indptr[b], a.num_pages};
  if (t < kWave) {
    const Walk w = qn > 0 ? tree_walk(a, qb, qn, path, dest + a.room, dest + 2 * a.room,
                                      dest + 3 * a.room)
                          : Walk{0, 0, -1};
    if (t == 0) walk = w;
  }
  __syncthreads();
  const int n = walk.length, still = walk.still;
  if (blockIdx.x == 0) {
    for (int i = t; i < qn; i += 256) a.path[qb + i] = i < n ? path[i] : -1;
    if (t == 0) {
      a.count[b] = n;
      a.next[b] = walk.last;
    }
    if (b == a.batch - 1)
      for (int i = max(a.q_indptr[a.batch], 0) + t; i < a.rows; i += 256) a.path[i] = -1;
  }
  if (still == n || cached < 0 || pages.count <= 0) return;  // (nothing to move, or no tables)
  for (int i = still + t; i < n; i += 256) {
    const int from = cached + path[i], to = cached + i;
    source[i] = pages.page_of(from) * kPage + from % kPage;
    dest[i] = pages.page_of(to) * kPage + to % kPage;
  }
  __syncthreads();
  constexpr int kBytes = kFp8 ? kFp8Page : kMoveBfPage;
  uint8_t* const data = a.cache + (size_t)blockIdx.x * a.num_pages * kBytes;
  auto page = [&](int slot) { return data + (size_t)(slot / kPage) * kBytes; };
  for (int i0 = still, m; i0 < n; i0 += m) {
    const int place = (cached + i0) % 4;  // of the lot's first row in its quad
    m = min(kMoveRows - place, n - i0);
    if constexpr (kFp8) {
      // v: a word (head, dim) of two heads a thread; k: 16 bytes of one row; a scale byte
      unsigned v[kMoveRows][2], w[2];
      const int to_v = dest[i0], kr = min(t >> 5, m - 1), ku = t & 31;
      unsigned* const dst = (unsigned*)(page(to_v) + fp8_v_at(t >> 6, to_v & 12, 0)) + (t & 63);
      w[0] = dst[0];
      w[1] = dst[kFp8Head];  // (four heads on)
#pragma unroll
      for (int r = 0; r < kMoveRows; ++r) {
        const int from = source[i0 + min(r, m - 1)];
        const unsigned* src =
            (const unsigned*)(page(from) + fp8_v_at(t >> 6, from & 12, 0)) + (t & 63);
        v[r][0] = src[0] >> 8 * (from & 3) & 255;
        v[r][1] = src[kFp8Head] >> 8 * (from & 3) & 255;
      }
      const int from = source[i0 + kr], to = dest[i0 + kr];
      const unsigned k_at = (ku >> 2) * kFp8Head + (ku & 3) * 16;
      const int scale_at = fp8_scale_at((ku >> 1) & 7, ku & 1, 0);
      const u32x4 k = *(const u32x4*)(page(from) + k_at + from % kPage * kFp8Row);
      const uint8_t scale = page(from)[scale_at + from % kPage];
      moe::wait_vmcnt<0>();
      __syncthreads();
#pragma unroll
      for (int r = 0; r < kMoveRows; ++r) {
        if (r >= m) break;
        const int bit = 8 * (place + r);
        w[0] = (w[0] & ~(255u << bit)) | v[r][0] << bit;
        w[1] = (w[1] & ~(255u << bit)) | v[r][1] << bit;
      }
      dst[0] = w[0];
      dst[kFp8Head] = w[1];
      if ((t >> 5) < m) {
        *(u32x4*)(page(to) + k_at + to % kPage * kFp8Row) = k;
        if (ku < 16) page(to)[scale_at + to % kPage] = scale;
      }
    } else {
      // 16 bytes of every other row a thread
      u32x4 w[kMoveRows / 2];
      const int first = t >> 7, u = t & 127;
      const unsigned at = (u >> 3) * kMoveBfHead + (u & 7) * 16;
#pragma unroll
      for (int r = 0; r < kMoveRows / 2; ++r) {
        const int from = source[i0 + min(first + 2 * r, m - 1)];
        w[r] = *(const u32x4*)(page(from) + at + from % kPage * (kD * 2));
      }
      moe::wait_vmcnt<0>();
      __syncthreads();
#pragma unroll
      for (int r = 0; r < kMoveRows / 2; ++r) {
        if (first + 2 * r >= m) break;
        const int to = dest[i0 + first + 2 * r];
        *(u32x4*)(page(to) + at + to % kPage * (kD * 2)) = w[r];
      }
    }
  }
}

// Pages copied in every layer: grid (pages, layers), four 16-byte loads of a thread in flight.  Bound by
// the bytes: 80 pages of the 8-bit cache in 36 layers, 96 MB read and written, 15.3 us;
// two pages in 24 layers 2.8 (3.3 with one load at a time).
__global__ __launch_bounds__(256) void copy_pages_kernel(uint8_t* __restrict__ cache,
                                                         int num_pages, int units,
                                                         const int* __restrict__ src,
                                                         const int* __restrict__ dst) {
  const int from = src[blockIdx.x], to = dst[blockIdx.x];
  if ((unsigned)from >= (unsigned)num_pages || (unsigned)to >= (unsigned)num_pages) return;
  u32x4* const data = (u32x4*)cache + (size_t)blockIdx.y * num_pages * units;
  const u32x4* const in = data + (size_t)from * units;
  u32x4* const out = data + (size_t)to * units;
  for (int i0 = threadIdx.x; i0 < units; i0 += 1024) {
    u32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = in[min(i0 + 256 * j, units - 1)];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + 256 * j < units) out[i0 + 256 * j] = x[j];
  }
}

}  // namespace attn

extern "C" {

int attn_launch_tree_commit(void* cache, int layers, int num_pages, bool fp8,
                            const int* page_indptr, const int* page_indices, const int* kv_len,
                            const int* q_indptr, int batch, int rows, int max_q_len,
                            const int* tokens, const int* parents, const int* chosen, int* path,
                            int* count, int* next, hipStream_t s) {
  const dim3 grid(layers, batch);
  // LDS for the trees at hand (room for 1024 nodes leaves a CU no more than 6 workgroups)
  const int room = std::min(max_q_len, attn::kMoveNodes);
  const size_t lds = (room <= attn::kWave ? 3 : 6) * sizeof(int) * room;
  const attn::CommitArgs a{(uint8_t*)cache, page_indptr, page_indices, kv_len, q_indptr, tokens,
                           parents, chosen, path, count, next, batch, rows, num_pages, room};
  if (fp8)
    hipLaunchKernelGGL(attn::tree_commit_kernel<true>, grid, dim3(256), lds, s, a);
  else
    hipLaunchKernelGGL(attn::tree_commit_kernel<false>, grid, dim3(256), lds, s, a);
  return hipGetLastError() == hipSuccess ? 0 : -6;
}

int attn_launch_copy_pages(void* cache, int layers, int num_pages, int page_bytes, const int* src,
                           const int* dst, int n, hipStream_t s) {
  hipLaunchKernelGGL(attn::copy_pages_kernel, dim3(n, layers), dim3(256), 0, s, (uint8_t*)cache,
                     num_pages, page_bytes / 16, src, dst);
  return hipGetLastError() == hipSuccess ? 0 : -6;
}

}  // extern "C"
