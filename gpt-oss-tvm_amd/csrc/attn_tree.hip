// Attention of trees of drafted tokens over the paged cache (gfx950), bf16 and 8-bit.
//
// A sequence of c cached tokens holds its tree's node i at index c + i of its pages; node i sees
// the cached keys (those of the window, where there is one) and the nodes that its mask has:
//   out = sum_j p_j v_j / (sum_j p_j + exp(sink)),  p_j = exp(sm_scale q . k_j)
// rounded to bf16 once; a node that sees no key gets 0.  Scores, sums and outputs in fp32,
// exponents in units of log2.
#include <stdint.h>

#include <type_traits>

#include "attn_common.h"

namespace attn {

constexpr int kHeadBytes = kPage * kD * 2;  // of a bf16 page's k or v of one head
constexpr int kBfPage = 2 * kHkv * kHeadBytes;
constexpr float kTreeLog2e = 1.4426950408889634f;
constexpr float kTreeMost = 16777216.0f;    // 2^24
constexpr int kTreeBlock = 64;              // keys
constexpr int kTreePart = 8 * kWave * 4;    // numbers of a wave's part
constexpr int kTreeHalf = kTreeBlock * kD * 2;  // bytes of a block's k or v in LDS

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4;
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

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
  // parts, as a wave's lanes hold them (rows of 16 bytes 256 bytes apart took twice the time):
  float* part_o;   // [workers + tiles][kv head][tokens of a tile / 4][8][lane][4]
  float* part_ml;  // [workers + tiles][kv head][tokens of a tile / 4][32 columns][2]
  int4* line;      // [batch][tiles]: first part, parts (0 or 1: none to merge), row, rows
  int words, num_pages, window, batch, tiles, workers, least, lead;
  float c2;        // sm_scale log2(e)
};

__device__ __forceinline__ f32x16 tree_mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

template <int kValue>
using Const = std::integral_constant<int, kValue>;

// The blocks of 64 keys that a sequence's nodes look at.
struct TreeSpan {
  int first, blocks;
  __device__ __forceinline__ TreeSpan(int cached, int total, int window) {
    // positions are at or past the cached tokens' end
    const int lo = window > 0 ? max(0, cached - window + 1) : 0;
    first = lo / kTreeBlock;
    blocks = total > lo ? (total - 1) / kTreeBlock - first + 1 : 0;
  }
};

// The work of a kv head in one line: the blocks of every tile of every sequence (up to 64, one a
// lane; a tile without keys counts as one), one after the other, cut into equal pieces of at least
// `least`, a worker each; before every tile but the first `lead` blocks that nobody has, for what
// beginning another tile costs.  Sequences of all lengths and few of them fill the chip alike, and
// it follows from the keys and not from the caller's bound on them, which only trims the workers.
// A worker's part of tile g (counted over all sequences) that it does not have whole goes to place
// worker + g of the workspace: two parts never share one, as one step in the line moves on
// to the next worker, the next tile or both.
struct TreeLine {
  int64_t before, after;  // the line up to the lane's sequence and with it
  int64_t all, piece;
  int blocks;             // of one of its tiles
  int tiles_before;       // of the sequences before it
  int row, nodes, total, page, pages;  // its tables
  TreeLine() = default;
  __device__ __forceinline__ TreeLine(const TreeArgs& a, int tokens) {
    const int lane = threadIdx.x & 63, b = min(lane, a.batch - 1);
    row = a.q_indptr[b];
    nodes = a.q_indptr[b + 1] - row;
    page = a.page_indptr[b];
    pages = a.page_indptr[b + 1] - page;
    total = a.kv_len[b];
    if (pages <= 0) total = 0;
    blocks = max(1, TreeSpan(max(total - nodes, 0), total, a.window).blocks);
    const int tiles = lane < a.batch ? min(max((nodes + tokens - 1) / tokens, 0), a.tiles) : 0;
    const int64_t mine = (int64_t)tiles * (a.lead + blocks);
    after = mine;
    int tiles_after = tiles;
    // (by register moves: within rows of 16 lanes, then across them; through LDS 0.4 us more)
    auto step = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
      auto moved = [&](int x) {
        return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xF,
                                           false);
      };
      const uint64_t low = (uint32_t)moved((int)(uint32_t)after);
      after += (int64_t)(low | (uint64_t)(uint32_t)moved((int)(after >> 32)) << 32);
      tiles_after += moved(tiles_after);
    };
    step(Const<0x111>(), Const<0xF>());  // row_shr:1, 2, 4, 8
    step(Const<0x112>(), Const<0xF>());
    step(Const<0x114>(), Const<0xF>());
    step(Const<0x118>(), Const<0xF>());
    step(Const<0x142>(), Const<0xA>());  // row_bcast:15 into rows 1 and 3
    step(Const<0x143>(), Const<0xC>());  // row_bcast:31 into rows 2 and 3
    before = after - mine;
    tiles_before = tiles_after - tiles;
    all = max((int64_t)0, lane_of(after, 63) - a.lead);  // (it begins at a.lead)
    // (exact: far below 2^53, and a quotient is an integer or 1 / workers away from the next)
    piece = max((int64_t)a.least, (int64_t)((double)(all + a.workers - 1) / (double)a.workers));
  }
  static __device__ __forceinline__ int64_t lane_of(int64_t x, int l) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, l) |
                     (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32);
  }
  // what the merge needs to know of the lane's sequence's tiles
  __device__ __forceinline__ void write(const TreeArgs& a, int tokens) const {
    const int b = threadIdx.x & 63, used = (nodes + tokens - 1) / tokens;
    if (b >= a.batch) return;
    for (int i = 0; i < a.tiles; ++i) {
      const int64_t from = before + (int64_t)i * (a.lead + blocks);  // (less lead: it begins there)
      // (exact, as above)
      const int first = (int)((double)from / (double)piece);
      const int last = (int)((double)(from + blocks - 1) / (double)piece);
      a.line[b * a.tiles + i] =
          i < used ? make_int4(first + tiles_before + i, last - first + 1, row + i * tokens,
                               min(tokens, nodes - i * tokens))
                   : make_int4(0, 0, 0, 0);
    }
  }
};

// o over the sum and the sink's share, at the reference point m (log2).  l is 0 only where no
// key was seen (or none with a score above -inf).
__device__ __forceinline__ float tree_share(float l, float m, uint16_t sink) {
  return l == 0.0f ? 0.0f
                   : 1.0f / (l + __builtin_amdgcn_exp2f(fmaf(bf2f(sink), kTreeLog2e, -m)));
}
// The weight of a partial state at the reference point `top`; one that saw no key: m = -inf, l = 0.
__device__ __forceinline__ float tree_weight(float m, float l, float top) {
  return m == -INFINITY && l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - top);
}

// A tile of 4 kC tokens x the 8 heads of a kv head, a wave 4 tokens (32 columns); kK groups of kC
// waves take every kK-th block of 64 keys.  A group stages its blocks through LDS as bf16, k in
// rows of 128 bytes whose 16-byte units are XORed with the row's bits 1 .. 3; v of a bf16 cache
// in rows too, read through the transposing LDS load, v of the 8-bit cache as the rows of
// V^T, whose operand order its pages have.
//  * S^T = K Q^T: lane (column l % 32, half h = l / 32) has the keys 8 (i / 4) + 4 h + i % 4 of a
//    32-key tile in elements i = 0 .. 15, which are, packed to bf16, the operands of two
//    products O^T += V^T P^T over 16 keys each.
//  * p enters as two bf16 pieces, off by 2^-16 of itself at most, as the framework's other
//    attention over few tokens or a bf16 cache has it; the sum takes both.  Tiles of 32 tokens of
//    the 8-bit cache round it once, as its long chunks do (a weight off by half a bf16 step at
//    most, where the cached values are off by up to 16 times as much): errors against 64 bits
//    0.0020 to 0.0021 instead of 0.0017, but two pieces would take 192 us instead of 132 for 2
//    trees of 26 over up to 131072, 49 instead of 40 for one of 64 over 16000.  What they cost
//    the others, graph replays, us with one and with two: 16 x 8 over 4000 29 and 32, 1 x 5
//    over 777 16.1 and 16.4, 32 x 16 in a window 17.0 and 17.4.
//  * No running maximum: the reference point is the maximum of the first keys that a column
//    sees, and is renewed only when a tile's sum passes 2^24.
//  * Blocks that every token of a wave sees whole take no mask; in the others (the tree's own, a
//    window's edge) a lane has its token's 32 bits of a tile, and tiles of which nobody sees a key
//    are passed over (32 trees of 16 nodes in a window 12.2 -> 10.9).
//
// What bounds it, with us of the kernel alone at four sizes: 1 tree of 5 nodes over 777 tokens, 16
// of 8 over up to 4000 (bf16), 1 of 64 over 16000, 2 of 26 over up to 131072 (8-bit): 8.7, 24,
// 32, 134.  (Comparisons below at 4 to 16 tokens are of probabilities in one piece.)
//  * Few nodes: the keys' bytes, and at the smallest calls the loads that wait for one another
//    (tables, page ids, keys, parts).  16 x 8: 80 MB, 3.4 TB/s; a copy reaches 5.0.
//  * Many nodes: the products and the exponentials beside them.  2 x 26: 85 GFLOP for tokens that
//    are there, 630 TFLOP/s of the 1280 that a large bf16 product reaches; a wave's 32 keys take
//    260 cycles of matrix instructions and 250 of others, 160 of them exponentials.  At 146 in
//    all it was 128 without the exponentials, 135 without the second product, 153 without
//    staging: no part carries it alone.  Two 32-key tiles at once, the operands of a tile read
//    ahead, four buffers and half the barriers, sums by additions and raised wave priorities were
//    each timed and gained nothing (144 .. 175).
//  * kC: a tile as wide as the tree, so that its keys are staged once, up to 32 tokens.  kK, with
//    as many waves on the chip, both launches: 8-token tiles of 2 and 4 groups, 16 x 8 25.5 and 28,
//    64 x 8 over up to 1000 34 and 41; 4-token tiles of 4 and 8, 64 x 4 over up to 500 24 and 30;
//    32-token tiles of 2 and 1, 2 x 26 153 and 160.
//  * Registers: up to 16 tokens 256 a lane (32 trees of 16 nodes in a window: 14 when this was
//    chosen; with 128, spilled, 21); 32 tokens take 16 waves and so 128.
template <int kC, int kK>
struct TreeLds {
  static constexpr int kBufs = kC == 1 ? 1 : 2;  // one wave needs no second buffer
  __align__(16) uint8_t tiles[kK][kBufs][2][kTreeHalf];
  float2 ml[kK][kC][32];
  int2 bad[kK][kC];  // a wave's first and last block with an infinity or a NaN in v (bf16)
};

// Blocks begin .. end - 1 of a tile whose sequence has qn nodes from row qb on and L tokens in all;
// the result goes to out, or where it is a part to `place` of the workspace.
template <bool kFp8, int kC, int kK>
__device__ __forceinline__ void tree_piece(const TreeArgs& a, TreeLds<kC, kK>& lds, int hk,
                                           const PageList& pages, int tile, int qb, int qn, int L,
                                           int begin, int end, int place) {
  constexpr int kBufs = TreeLds<kC, kK>::kBufs;
  constexpr int kUnits = (kFp8 ? 8 : 16) / kC;  // 1 KB loads of a block that a wave makes
  constexpr int kPieces = kFp8 && kC == 8 ? 1 : 2;  // of p
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));  // (what follows from it is not carried over to the next piece)
  const int lane = t & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6), cw = wave % kC, kg = wave / kC;
  const int t0 = tile * 4 * kC, nt = min(4 * kC, qn - t0), row0 = qb + t0;
  const int cached = max(L - qn, 0);
  const bool active = 4 * cw < nt;
  const int last_page = max(0, min(pages.count - 1, (L - 1) / kPage));
  const int steps = (end - begin + kK - 1) / kK;  // of every group
  constexpr int kPageSize = kFp8 ? kFp8Page : kBfPage;

  // Staging.  The group's i-th block is begin + kg + kK i; lane 4 j + p holds its page p for
  // the j-th of 16 blocks.
  int ids = 0;
  auto fetch_ids = [&](int i) {
    const int page = (begin + kg + kK * (i + (lane >> 2))) * 4 + (lane & 3);
    ids = pages.clamp(pages.ids[min(page, last_page)]);
  };
  struct Raw {
    u32x4 data[kUnits];
    uint32_t ks[kFp8 ? kUnits : 1], vs[kFp8 ? kUnits : 1];
  };
  // unit u of the wave: load u kC + cw of the block: bf16 [k, v][page][half of its rows], 8-bit
  // [k, v][page]
  auto load = [&](Raw& x, int i) __attribute__((always_inline)) {
    if ((i & 15) == 0 && i > 0) fetch_ids(i);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int id = u * kC + cw;
      const int p = kFp8 ? id & 3 : (id >> 1) & 3, kv = kFp8 ? id >> 2 : id >> 3;
      const uint8_t* page = a.cache + (size_t)(unsigned)__builtin_amdgcn_readlane(
                                          ids, 4 * (i & 15) + p) * kPageSize;
      if constexpr (kFp8) {
        x.data[u] = *(const u32x4*)(page + (kv ? kFp8V : 0) + hk * kFp8Head + lane * 16);
        const uint8_t* s = page + kFp8Scales + hk * 2 * kPage + (lane >> 4) * 4;
        if (!kv) x.ks[u] = *(const uint32_t*)s;
        x.vs[u] = *(const uint32_t*)(s + kPage);
      } else {
        x.data[u] = *(const u32x4*)(page + (kv * kHkv + hk) * kHeadBytes + (id & 1) * 1024 +
                                    lane * 16);
      }
    }
  };
  int2 bad = make_int2(INT32_MAX, -1);
  auto store = [&](Raw& x, uint8_t* kt, uint8_t* vt, int i) __attribute__((always_inline)) {
    const int kb = (begin + kg + kK * i) * kTreeBlock;
    if constexpr (!kFp8) {
      uint32_t full = 0u;  // bits 15 and 31: an exponent of all ones
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
        if ((u * kC + cw) >> 3)
#pragma unroll
          for (int j = 0; j < 4; ++j) full |= (x.data[u][j] & 0x7F807F80u) + 0x00800080u;
      if (__any(full & 0x80008000u)) {
        bad = make_int2(min(bad.x, i), i);
        if (lane == 0) lds.bad[kg][cw] = bad;
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
          if ((u * kC + cw) >> 3)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t y = x.data[u][j];
              x.data[u][j] = ((y & 0x7F80u) == 0x7F80u ? 0u : y & 0xFFFFu) |
                             ((y & 0x7F800000u) == 0x7F800000u ? 0u : y & 0xFFFF0000u);
            }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int id = u * kC + cw;
      const int p = kFp8 ? id & 3 : (id >> 1) & 3, kv = kFp8 ? id >> 2 : id >> 3;
      if constexpr (!kFp8) {
        const int key = kPage * p + 8 * (id & 1) + (lane >> 3), part = lane & 7;
        const int at = kv ? part ^ ((key & 2) << 1) : part ^ ((key >> 1) & 7);
        *(u32x4*)((kv ? vt : kt) + key * 128 + (at << 4)) = x.data[u];
      } else if (!kv) {
        // 16 dims of key lane / 4; a row that must not be used (255) is NaN in k and 0 in v
        const int byte = 8 * ((lane >> 2) & 3), key = kPage * p + (lane >> 2);
        const uint32_t sk = (x.ks[u] >> byte) & 255u, sv = (x.vs[u] >> byte) & 255u;
        const bool bad = max(sk, sv) == kFp8BadScale;
        const float scale = __uint_as_float(min(sk, kFp8BadScale - 1u) << 23);
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = bad ? kFp8NanCodes : x.data[u][j];
        uint8_t* row = kt + key * 128;
        const int swz = (key >> 1) & 7, at = 2 * (lane & 3);
        *(bf16x8*)(row + ((at ^ swz) << 4)) = fp8_to_bf16(w[0], w[1], scale);
        *(bf16x8*)(row + (((at + 1) ^ swz) << 4)) = fp8_to_bf16(w[2], w[3], scale);
      } else {
        // four keys (quad lane / 16 of the page) of the dims r, 16 + r, 32 + r, 48 + r.  A 16-byte
        // unit of V^T's rows holds two quads: 4 m + h' and 4 m + 2 + h' for the product m of a
        // 32-key tile and the lanes' half h'.
        const int quad = 4 * p + (lane >> 4), r = lane & 15, n = quad & 7;
        const int unit = 4 * (quad >> 3) + 2 * (n >> 2) + (n & 1), part = (n >> 1) & 1;
        uint32_t keep = ~0u;
        if (kb + kTreeBlock > L) {  // stale codes past the sequence's end may be NaN
          const int m = min(max(L - (kb + 4 * quad), 0), 4);
          keep = m == 4 ? ~0u : (1u << (8 * m)) - 1u;
        }
        float s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s[j] = __uint_as_float(min((x.vs[u] >> (8 * j)) & 255u, kFp8BadScale - 1u) << 23);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
          const uint32_t w = x.data[u][dt] & keep;
          const auto a0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s[0], false);
          const auto a1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s[1], false);
          const auto a2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s[2], true);
          const auto a3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s[3], true);
          const uint32_t p0 = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, a1),
                                                    __builtin_bit_cast(uint32_t, a0), 0x07060100u);
          const uint32_t p1 = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, a3),
                                                    __builtin_bit_cast(uint32_t, a2), 0x07060100u);
          const int d = 16 * dt + r;
          *(uint2*)(vt + d * 128 + ((unit ^ ((d >> 1) & 7)) << 4) + 8 * part) = make_uint2(p0, p1);
        }
      }
    }
  };

  // whether the group has an i-th block; the first blocks' loads and q are on their way at once
  auto mine = [&](int i) { return begin + kg + kK * i < end; };
  Raw raw;
  if (mine(0)) {
    fetch_ids(0);
    load(raw, 0);
  }
  const int token = min(4 * cw + (c >> 3), nt - 1), row = row0 + token;
  const uint16_t sink = a.sinks[hk * kGroup + (c & 7)];
  const int pos = max(a.positions[row], cached);
  const uint32_t* const bits = a.mask + (size_t)row * a.words;
  const uint32_t bits0 = bits[0], bits1 = a.words > 1 ? bits[1] : 0u;  // most trees' all
  bf16x8 qv[4];
  {
    const u32x4* src = (const u32x4*)(a.q + ((size_t)row * kHq + hk * kGroup + (c & 7)) * kD);
#pragma unroll
    for (int s = 0; s < 4; ++s) qv[s] = moe::as_bf16x8(src[2 * s + h]);
  }
  // the furthest position of the wave's tokens: where a window begins that all of them see
  int far = max(pos, __shfl_xor(pos, 8, kWave));
  far = __builtin_amdgcn_readfirstlane(max(far, __shfl_xor(far, 16, kWave)));
  const int seen_from = a.window > 0 ? far - a.window : -1;  // the last key that not all see

  // The lane's token's bits of the keys k0 .. k0 + 31
  auto seen = [&](int k0) {
    auto first_of = [](int n) { return n >= 32 ? ~0u : (1u << max(n, 0)) - 1u; };
    auto word = [&](int w) {
      return w == 0 ? bits0 : w == 1 ? bits1 : w < a.words ? bits[w] : 0u;
    };
    const int from = k0 - cached;  // the first key's node
    const int lowest = a.window > 0 ? pos - a.window + 1 : 0;  // position
    uint32_t nodes = 0u;
    if (from >= 0) {
      const int w = from >> 5, s = from & 31;
      nodes = word(w) >> s;
      if (s) nodes |= word(w + 1) << (32 - s);
    } else if (from > -32) {
      nodes = bits0 << -from;
    }
    nodes &= first_of(L - k0);
    if (lowest > cached) {  // nodes before the window: a window shorter than the tree
      for (uint32_t left = nodes; left; left &= left - 1u) {
        const int i = __builtin_ctz(left);
        if (max(a.positions[qb + from + i], cached) < lowest) nodes &= ~(1u << i);
      }
    }
    return (first_of(cached - k0) & ~first_of(lowest - k0)) | nodes;
  };

  f32x16 o[2];
  bool fresh = true;  // no tile yet
  float mneg = INFINITY, l = 0.f;  // minus the column's reference point (not set: inf)
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  const moe::bf16x2 ones = {(__bf16)1.0f, (__bf16)1.0f};

  // where the lane reads in a block's tiles: k of its key c, step st at ^ 32 st; v of the 8-bit
  // cache of its dim c, product m and 32-key tile n at ^ (32 m + 64 n); of a bf16 cache the quarter
  // i % 4 of 16 dims of key i / 4 of four (i = lane % 16), the upper 32 dims at ^ 64
  const int k_at = c * 128 + ((h ^ ((c >> 1) & 7)) << 4);
  const int v_at = kFp8 ? k_at
                        : (4 * h + ((lane >> 2) & 3)) * 128 + ((lane >> 4) & 1) * 32 +
                              (lane & 3) * 8 + ((lane >> 3) & 1) * 64;
  // the 32 keys from 32 kt32 of a block on
  auto keys32 = [&](auto masked, const uint8_t* kt, const uint8_t* vt, int kb, int kt32)
      __attribute__((always_inline)) {
    constexpr bool kMasked = decltype(masked)::value;
    f32x16 s;
    uint32_t see = ~0u;
    if constexpr (kMasked) {
      see = seen(kb + 32 * kt32);
      if (!__any(see != 0u)) return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      const bf16x8 ka = *(const bf16x8*)(kt + 4096 * kt32 + (k_at ^ (32 * st)));
      s = tree_mfma(ka, qv[st], s);
    }
    if constexpr (kMasked) {
      const uint32_t mine = see >> (4 * h);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t keep = __builtin_amdgcn_sbfe((int)mine, 8 * (i >> 2) + (i & 3), 1);
        s[i] = __uint_as_float((keep & __float_as_uint(s[i])) | (~keep & 0xFF800000u));
      }
    }
    moe::bf16x2 p[kPieces][8];
    float ps;
    auto exps = [&](float mn) __attribute__((always_inline)) {
      ps = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e0 = __builtin_amdgcn_exp2f(fmaf(s[2 * i], a.c2, mn));
        const float e1 = __builtin_amdgcn_exp2f(fmaf(s[2 * i + 1], a.c2, mn));
        p[0][i] = moe::bf16x2{(__bf16)e0, (__bf16)e1};
        ps = __builtin_amdgcn_fdot2_f32_bf16(p[0][i], ones, ps, false);
        if constexpr (kPieces == 2) {
          p[1][i] = moe::bf16x2{(__bf16)(e0 - (float)p[0][i][0]), (__bf16)(e1 - (float)p[0][i][1])};
          ps = __builtin_amdgcn_fdot2_f32_bf16(p[1][i], ones, ps, false);
        }
      }
    };
    if (!fresh) exps(mneg);
    if (fresh || __any(!(ps < kTreeMost))) {
      float mx = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
      const uint32_t u = __float_as_uint(mx);
      const auto x = __builtin_amdgcn_permlane32_swap(u, u, false, false);
      mx = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
      const float m = -mneg, mn = fmaxf(m, mx * a.c2);
      const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      if (!fresh)
#pragma unroll
        for (int dt = 0; dt < 2; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
      l *= alpha;
      fresh = false;
      mneg = -mn;
      exps(mn == -INFINITY ? 0.0f : -mn);
    }
    l += ps;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      bf16x8 pb[kPieces];
#pragma unroll
      for (int n = 0; n < kPieces; ++n)
#pragma unroll
        for (int j = 0; j < 8; ++j) pb[n][j] = p[n][4 * m + (j >> 1)][j & 1];
#pragma unroll
      for (int dt = 0; dt < 2; ++dt) {
        bf16x8 va;
        if constexpr (kMasked && kC > 4) __builtin_amdgcn_sched_barrier(0);  // (registers)
        if constexpr (kFp8) {
          va = *(const bf16x8*)(vt + 4096 * dt + (v_at ^ (32 * m + 64 * kt32)));
        } else {
          u32x4 w;  // dim c of 32 dt of the keys 16 m + 8 j + 4 h ..
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const s16x4 four = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4)(vt + 4096 * kt32 + 2048 * m + 1024 * j + (v_at ^ (64 * dt))));
            const uint2 pair = __builtin_bit_cast(uint2, four);
            w[2 * j] = pair.x;
            w[2 * j + 1] = pair.y;
          }
          va = moe::as_bf16x8(w);
        }
#pragma unroll
        for (int n = 0; n < kPieces; ++n) o[dt] = tree_mfma(va, pb[n], o[dt]);
      }
    }
  };
  auto compute = [&](auto masked, int buf, int i) __attribute__((always_inline)) {
    const int kb = (begin + kg + kK * i) * kTreeBlock;
    const uint8_t *kt = lds.tiles[kg][buf][0], *vt = lds.tiles[kg][buf][1];
    if constexpr (decltype(masked)::value) {
#pragma unroll 1  // (registers)
      for (int kt32 = 0; kt32 < 2; ++kt32) keys32(masked, kt, vt, kb, kt32);
    } else {
      keys32(masked, kt, vt, kb, 0);
      keys32(masked, kt, vt, kb, 1);
    }
  };
  auto put = [&](int buf, int i) __attribute__((always_inline)) {
    store(raw, lds.tiles[kg][buf][0], lds.tiles[kg][buf][1], i);
  };
  // Infinities and NaN in v of a bf16 cache.  They must not meet the probability 0 of who does not
  // see their key, nor the second piece of one, which may be 0 or negative: staged as 0, they
  // go in behind the loop (blocks first to last of the group, again from memory) by products of
  // their own.  The largest number for them and for who sees them, whose square is past fp32's
  // range: +inf and NaN by one, -inf and NaN by another.  (At the products, in a branch of masked blocks,
  // they took registers of every call: 64 x 26 over 500 73 us and not 52, 2 x 26 over 40000 119
  // and not 79.)
  auto add_bad = [&](int first, int last) __attribute__((always_inline)) {
#pragma unroll 1
    for (int at = 4 * first; at < 4 * last + 4; ++at) {  // 16 keys, a page, at a time
      const int k0 = (begin + kg + kK * (at >> 2)) * kTreeBlock + kPage * (at & 3);
      const uint8_t* const page =
          a.cache +
          (size_t)(unsigned)pages.clamp(pages.ids[min(k0 / kPage, last_page)]) * kPageSize +
          (kHkv + hk) * kHeadBytes;
      const uint32_t see = seen(k0);
      const __bf16 big = (__bf16)3.3895314e38f, none = (__bf16)0.0f;
#pragma unroll
      for (int dt = 0; dt < 2; ++dt) {
        uint32_t x[8];
        bf16x8 marks, who;
        bool any = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = 8 * (j >> 2) + 4 * h + (j & 3);
          x[j] = *(const uint16_t*)(page + key * (kD * 2) + (32 * dt + c) * 2);
          any |= (x[j] & 0x7F80u) == 0x7F80u;
          who[j] = see >> key & 1u ? big : none;
        }
        if (!__any(any)) continue;
#pragma unroll
        for (int sign = 0; sign < 2; ++sign) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const bool is = (x[j] & 0x7FFFu) > 0x7F80u || x[j] == (sign ? 0xFF80u : 0x7F80u);
            marks[j] = is ? sign ? -big : big : none;
          }
          f32x16 inf;
#pragma unroll
          for (int i = 0; i < 16; ++i) inf[i] = 0.f;
          inf = tree_mfma(marks, who, inf);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[dt][i] += inf[i];
        }
      }
    }
  };

  // every load before the loop (the first block, q, the mask) done: the compiler then waits for
  // nothing but the next block there
  moe::wait_vmcnt<0>();
  if (!kFp8 && lane == 0) lds.bad[kg][cw] = bad;
  if (mine(0)) put(0, 0);
  if (mine(1)) load(raw, 1);
  if constexpr (kC > 1) moe::lds_barrier();
  int i = 0;
  auto run = [&](auto masked, int to) __attribute__((always_inline)) {
    for (; i < to; ++i) {
      const int buf = kBufs == 1 ? 0 : i & 1, next = kBufs == 1 ? 0 : buf ^ 1;
      if (active && mine(i)) compute(masked, buf, i);
      if (mine(i + 1)) put(next, i + 1);
      if (mine(i + 2)) load(raw, i + 2);  // in flight during the next block's products
      if constexpr (kC > 1) moe::lds_barrier();
    }
  };
  // steps whose block every token of the wave sees whole: from whole0 to whole1
  auto step_of = [&](int block) {
    return min(max((block - begin - kg + kK - 1) / kK, 0), steps);
  };
  const int whole1 = step_of(max(cached / kTreeBlock, begin));
  const int window0 = seen_from >= 0 ? seen_from / kTreeBlock + 1 : 0;
  const int whole0 = min(whole1, step_of(max(window0, begin)));
  run(std::true_type{}, whole0);
  run(std::false_type{}, whole1);
  run(std::true_type{}, steps);

  if constexpr (!kFp8) {
    if (active) {
#pragma unroll
      for (int w = 0; w < kC; ++w) {
        const int2 other = lds.bad[kg][w];
        bad = make_int2(min(bad.x, other.x), max(bad.y, other.y));
      }
      const int first = __builtin_amdgcn_readfirstlane(bad.x);
      const int last = __builtin_amdgcn_readfirstlane(bad.y);
      if (last >= 0) add_bad(first, last);
    }
  }
  float lt = l + __shfl_xor(l, 32, kWave);
  if constexpr (kK > 1) {
    // the groups' states into the first group's, in order, through the tiles' LDS
    if constexpr (kC == 1) moe::lds_barrier();  // every wave is done with its tile
    f32x4* const part = (f32x4*)&lds.tiles[0][0][0][0] + cw * 8 * kWave + lane;
    if (kg > 0) {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        part[((kg - 1) * kC * 8 + q) * kWave] =
            f32x4{o[q >> 2][4 * (q & 3)], o[q >> 2][4 * (q & 3) + 1],
                  o[q >> 2][4 * (q & 3) + 2], o[q >> 2][4 * (q & 3) + 3]};
      if (h == 0) lds.ml[kg][cw][c] = make_float2(-mneg, lt);
    }
    moe::lds_barrier();
    if (kg > 0) return;
    float top = -mneg;
#pragma unroll
    for (int g = 1; g < kK; ++g) top = fmaxf(top, lds.ml[g][cw][c].x);
    const float w0 = tree_weight(-mneg, lt, top);
    lt *= w0;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] *= w0;
#pragma unroll
    for (int g = 1; g < kK; ++g) {
      const float2 other = lds.ml[g][cw][c];
      const float w = tree_weight(other.x, other.y, top);
      lt = fmaf(other.y, w, lt);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const f32x4 po = part[((g - 1) * kC * 8 + q) * kWave];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[q >> 2][4 * (q & 3) + j] = fmaf(po[j], w, o[q >> 2][4 * (q & 3) + j]);
      }
    }
    mneg = -top;
  }
  if (4 * cw + (c >> 3) >= nt) return;
  if (place < 0) {
    const float f = tree_share(lt, -mneg, sink);
    uint16_t* const out = a.out + ((size_t)row * kHq + hk * kGroup + (c & 7)) * kD;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        uint16_t v4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v4[j] = f2bf(o[dt][i + j] * f);
        *(uint2*)(out + 32 * dt + 2 * i + 4 * h) =
            make_uint2((uint32_t)v4[0] | ((uint32_t)v4[1] << 16),
                       (uint32_t)v4[2] | ((uint32_t)v4[3] << 16));
      }
  } else {
    const size_t at = ((size_t)place * kHkv + hk) * kC + cw;
#pragma unroll
    for (int q = 0; q < 8; ++q)
      *(f32x4*)(a.part_o + at * kTreePart + (q * kWave + lane) * 4) =
          f32x4{o[q >> 2][4 * (q & 3)], o[q >> 2][4 * (q & 3) + 1], o[q >> 2][4 * (q & 3) + 2],
                o[q >> 2][4 * (q & 3) + 3]};
    if (h == 0) *(float2*)(a.part_ml + (at * 32 + c) * 2) = make_float2(-mneg, lt);
  }
}

template <bool kFp8, int kC, int kK>
__global__ __launch_bounds__(64 * kC * kK)
__attribute__((amdgpu_waves_per_eu(kC <= 4 ? 2 : 4))) void tree_kernel(TreeArgs a) {
  __shared__ TreeLds<kC, kK> lds;
  __shared__ TreeLine lines[kWave];  // (out of the registers)
  // x: (worker, kv head); without workers (sequence, tile, kv head)
  const int hk = blockIdx.x % kHkv, worker = blockIdx.x / kHkv, lane = threadIdx.x & 63;
  int64_t at = 0, stop = 1;
  if (a.workers > 0) {
    const TreeLine line(a, 4 * kC);
    const int64_t piece = TreeLine::lane_of(line.piece, 0);
    at = worker * piece + a.lead;
    stop = min(at + piece, line.all + a.lead);
    if (blockIdx.x == 0 && threadIdx.x < kWave) line.write(a, 4 * kC);
    if (at >= stop) return;
    if (threadIdx.x < kWave) lines[lane] = line;
    moe::lds_barrier();
  }
  do {
    int tile = worker % a.tiles, first = 0, place = -1, qb, qn, L, page, pages;
    int64_t n = INT32_MAX;
    if (a.workers > 0) {
      const TreeLine& line = lines[__builtin_ctzll(__ballot(lines[lane].after > at))];
      auto one = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
      const int blocks = one(line.blocks);
      const int from = (int)(at - TreeLine::lane_of(line.before, 0));
      tile = from / (a.lead + blocks);
      first = from - tile * (a.lead + blocks) - a.lead;
      if (first < 0) {  // the blocks before a tile
        at -= first;
        if (at >= stop) return;
        first = 0;
      }
      n = min((int64_t)(blocks - first), stop - at);
      if (n < blocks) place = worker + one(line.tiles_before) + tile;
      qb = one(line.row);
      qn = one(line.nodes);
      L = one(line.total);
      page = one(line.page);
      pages = one(line.pages);
    } else {
      const int b = worker / a.tiles;
      qb = a.q_indptr[b];
      qn = a.q_indptr[b + 1] - qb;
      if (tile * 4 * kC >= qn) return;
      page = a.page_indptr[b];
      pages = a.page_indptr[b + 1] - page;
      L = pages > 0 ? a.kv_len[b] : 0;
    }
    const TreeSpan span(max(L - qn, 0), L, a.window);
    tree_piece<kFp8, kC, kK>(a, lds, hk, PageList{a.page_indices + page, pages, a.num_pages}, tile,
                             qb, qn, L, span.first + first,
                             span.first + (int)min(first + n, (int64_t)span.blocks), place);
    at += n;
    if (at < stop) moe::lds_barrier();  // the next piece's tiles go where this one's parts lie
  } while (at < stop);
}

// The parts of a tile merged, in order: a wave a quarter of a half (q) of a wave's 4 tokens of a kv
// head, in the lanes that wrote them; eight parts' loads in flight.  `tokens`: of a tile.
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a, int tokens) {
  const int waves = tokens / 4, lane = threadIdx.x & 63, c = lane & 31;
  const int group = blockIdx.y >> 1, hk = group / waves, cw = group % waves;
  const int q = 4 * (blockIdx.y & 1) + (threadIdx.x >> 6);
  const int token = 4 * cw + (c >> 3), head = hk * kGroup + (c & 7);
  const int d = 32 * (q >> 2) + 8 * (q & 3) + 4 * (lane >> 5);
  const int4 tile = a.line[blockIdx.x];
  const int used = tile.y;
  if (used <= 1 || token >= tile.w) return;  // (written already, or no token)
  const size_t step = (size_t)kHkv * waves, at = tile.x * step + group;
  float m = -INFINITY, l = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < used; s0 += 8) {
    float2 ml[8];
    f32x4 po[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const size_t pt = at + (size_t)min(s0 + j, used - 1) * step;
      ml[j] = *(const float2*)(a.part_ml + (pt * 32 + c) * 2);
      po[j] = *(const f32x4*)(a.part_o + pt * kTreePart + (q * kWave + lane) * 4);
    }
    float mn = m;
#pragma unroll
    for (int j = 0; j < 8; ++j) mn = s0 + j < used ? fmaxf(mn, ml[j].x) : mn;
    const float alpha = tree_weight(m, l, mn);
    l *= alpha;
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] *= alpha;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (s0 + j >= used) continue;
      const float w = tree_weight(ml[j].x, ml[j].y, mn);
      l = fmaf(ml[j].y, w, l);
#pragma unroll
      for (int q = 0; q < 4; ++q) o[q] = fmaf(po[j][q], w, o[q]);
    }
    m = mn;
  }
  const float f = tree_share(l, m, a.sinks[head]);
  uint16_t v4[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) v4[q] = f2bf(o[q] * f);
  *(uint2*)(a.out + ((size_t)(tile.z + token) * kHq + head) * kD + d) =
      make_uint2((uint32_t)v4[0] | ((uint32_t)v4[1] << 16),
                 (uint32_t)v4[2] | ((uint32_t)v4[3] << 16));
}

}  // namespace attn

extern "C" {

// tokens: of a tile, 4, 8, 16 or 32; workers: of a kv head, 0: a workgroup a tile (more than 64
// sequences); else part_o of 64 x 64 and part_ml of 64 x 2 numbers for each token of
// workers + batch * tiles tiles, and line of 16 bytes for each of batch * tiles.
int attn_launch_tree(const void* q, const int* q_indptr, int batch, int max_q_len,
                     const void* mask, int words, const int* positions, const void* cache,
                     bool fp8, const int* page_indptr, const int* page_indices, int num_pages,
                     const int* kv_len, int window, float sm_scale, const void* sinks, void* out,
                     int tokens, int workers, int least, int lead, float* part_o, float* part_ml,
                     void* line, hipStream_t s) {
  if (workers < 0 || (workers > 0 && batch > 64) || least < 1) return -6;
  const int tiles = (max_q_len + tokens - 1) / tokens;
  const attn::TreeArgs a{(const uint16_t*)q, q_indptr, (const uint32_t*)mask, positions,
                         (const uint8_t*)cache, page_indptr, page_indices, kv_len,
                         (const uint16_t*)sinks, (uint16_t*)out, part_o, part_ml, (int4*)line, words,
                         num_pages, window, batch, tiles, workers, least, lead,
                         sm_scale * attn::kTreeLog2e};
  const int grid = attn::kHkv * (workers > 0 ? workers : batch * tiles);
  auto go = [&](auto kernel, int waves) {
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * waves), 0, s, a);
  };
  if (tokens == 4)
    fp8 ? go(attn::tree_kernel<true, 1, 4>, 4) : go(attn::tree_kernel<false, 1, 4>, 4);
  else if (tokens == 8)
    fp8 ? go(attn::tree_kernel<true, 2, 2>, 4) : go(attn::tree_kernel<false, 2, 2>, 4);
  else if (tokens == 16)
    fp8 ? go(attn::tree_kernel<true, 4, 2>, 8) : go(attn::tree_kernel<false, 4, 2>, 8);
  else if (tokens == 32)
    fp8 ? go(attn::tree_kernel<true, 8, 2>, 16) : go(attn::tree_kernel<false, 8, 2>, 16);
  else
    return -6;
  if (hipGetLastError() != hipSuccess) return -6;
  if (workers > 0)
    hipLaunchKernelGGL(attn::tree_merge_kernel, dim3(batch * tiles, attn::kHkv * tokens / 2),
                       dim3(256), 0, s, a, tokens);
  return hipGetLastError() == hipSuccess ? 0 : -6;
}

}  // extern "C"
