// Shapes, page tables and the 8-bit cache format shared by the attention kernels.
#pragma once

#include "moe_common.h"

namespace attn {

using moe::bf16x8;
using moe::bf2f;
using moe::f2bf;
using moe::f32x4;
using moe::kWave;
using moe::load_dev;
using moe::store_dev;
using moe::u32x4;

constexpr int kD = 64;          // head_dim
constexpr int kHq = 64;         // query heads
constexpr int kHkv = 8;         // key/value heads
constexpr int kGroup = kHq / kHkv;
constexpr int kPage = 16;       // tokens per page
constexpr int kQkvHeads = kHq + 2 * kHkv;

// A sequence's page list: the page holding position pos.  The list index is
// clamped to the sequence's pages and the page id to the pool, so a page table
// that does not cover kv_len reads wrong keys instead of foreign memory (the
// host sizes the tables; this only keeps a bad table from faulting).
struct PageList {
  const int* ids;
  int count, pool;
  // a table entry clamped into the pool (callers that read entries ahead
  // clamp them at use)
  __device__ __forceinline__ int clamp(int id) const { return min(max(id, 0), pool - 1); }
  __device__ __forceinline__ int page_of(int pos) const {
    return clamp(ids[max(min(pos / kPage, count - 1), 0)]);
  }
};

// max of x over lanes l, l ^ 16, l ^ 32, l ^ 48 (the four 16-lane rows) in
// registers: swapping x with itself, v_permlane32_swap returns x of lanes
// l & 31 and l | 32, v_permlane16_swap x of rows 2 (l / 32) and 2 (l / 32) + 1
__device__ __forceinline__ float group_max(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float y = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(y), __float_as_uint(y), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ f32x4 mfma_bf16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// The 8-bit cache.  A row is the 64 values of one token, kv head and k or v:
// e4m3 codes and one scale byte s; code c stands for c 2^(s - 127).  With e the
// biased exponent of the row's largest magnitude, s = max(e - 7, 10): codes stay
// at or below 256 (the largest is never cut off, as it may be where it is scaled
// up to the format's 448), a power of two moves no value's rounding, and
// every nonzero code's value is 2^-126 or more, normal in bf16.  (At s = 247, the
// last, codes stop at 240: 256 would stand for 2^128.)  A row with an
// infinity or a NaN has s = 255 and stands for NaN: its codes are NaN in k, whose
// scores then are NaN for the queries that see the key and masked for the
// others, and 0 in v, which a matrix product multiplies by the probability 0
// of queries that do not see it.
//
// A page of 16 tokens and 8 kv heads is one record of 16640 bytes (a multiple of
// 128), half a bf16 page:
//   0      k codes  [head][token][dim]
//   8192   v codes  [head][token / 4][dim % 16][dim / 16][token % 4]
//   16384  scales   [head][k, v][token]
// v's order is the operand order of the matrix products over keys: a 16-byte
// unit holds four keys of the dims r, 16 + r, 32 + r and 48 + r, the rows r
// of four 16-row (or 32-row) tiles of V^T, so that no kernel transposes v.
constexpr int kFp8Row = kD;                       // bytes of a row's codes
constexpr int kFp8Head = kPage * kD;              // code bytes of a (page, k or v, head)
constexpr int kFp8V = kHkv * kFp8Head;            // where v's codes begin
constexpr int kFp8Scales = 2 * kHkv * kFp8Head;   // where the scales begin
constexpr int kFp8Page = kFp8Scales + 2 * kHkv * kPage;
constexpr uint32_t kFp8MinScale = 10, kFp8BadScale = 255;
constexpr uint32_t kFp8NanCodes = 0x7F7F7F7Fu;

// the page of a slot, or nullptr outside the pool
__device__ __forceinline__ uint8_t* fp8_page(uint8_t* cache, int slot, int num_pages) {
  if (slot < 0 || slot >= num_pages * kPage) return nullptr;
  return cache + (size_t)(slot / kPage) * kFp8Page;
}
// offset within a page of v's code of (head, token, dim)
__device__ __forceinline__ int fp8_v_at(int head, int token, int dim) {
  return kFp8V + head * kFp8Head + (token >> 2) * 256 + (dim & 15) * 16 + (dim >> 4) * 4 +
         (token & 3);
}
__device__ __forceinline__ int fp8_scale_at(int head, int kv, int token) {
  return kFp8Scales + (head * 2 + kv) * kPage + token;
}

// v's codes and the scales lie four tokens to a word.  Kernels that go over tokens by
// their slots take them in runs: a run begins at a multiple of four, or where a slot does
// not follow the one before, so a run of four is a quad whose words one wave moves
// whole, whatever the tokens' order and wherever sequences begin; shorter ones go byte by
// byte.  A wave or workgroup takes the runs that begin at tokens first .. first + 3.
struct SlotRuns {
  uint32_t begins;  // bit t: a run begins at token first + t (or there is no such token)
  __device__ __forceinline__ SlotRuns(const int* __restrict__ slots, int first, int n) {
    uint32_t slot[8];  // of the tokens first - 1 .. first + 6
#pragma unroll
    for (int t = 0; t < 8; ++t) slot[t] = (uint32_t)slots[min(max(first - 1 + t, 0), n - 1)];
    begins = 0;
#pragma unroll
    for (int t = 0; t < 7; ++t) {
      const bool follows = first + t > 0 && first + t < n && slot[t + 1] % 4 != 0 &&
                           slot[t + 1] == slot[t] + 1;
      begins |= (follows ? 0u : 1u) << t;
    }
  }
  // length (1 to 4) of the run that begins at token first + t
  __device__ __forceinline__ int length(int t) const {
    return __builtin_ctz(begins >> (t + 1) | 8u) + 1;
  }
};
// whether a run of `length` tokens from `slot` on is a quad of the pool
__device__ __forceinline__ bool fp8_quad(int slot, int length, int num_pages) {
  return length == 4 && slot >= 0 && slot < num_pages * kPage;
}

// Four words of four bytes, transposed.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
  const uint32_t ab = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u);
  const uint32_t cd = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  const uint32_t ab2 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
  const uint32_t cd2 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(cd, ab, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(cd, ab, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(cd2, ab2, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(cd2, ab2, 0x07060302u);
}

// scale byte of a row whose largest magnitude has the bf16 bits `top`
__device__ __forceinline__ uint32_t fp8_scale_of(uint32_t top) {
  const uint32_t e = top >> 7;
  return e == 255u ? kFp8BadScale : max(e, 7u + kFp8MinScale) - 7u;
}
// 2^(127 - s), s <= 247
__device__ __forceinline__ float fp8_inverse(uint32_t s) {
  return __uint_as_float((254u - min(s, 247u)) << 23);
}

// Two bf16 pairs of a row of scale byte s -> four codes.
__device__ __forceinline__ uint32_t fp8_codes(uint32_t a, uint32_t b, uint32_t s, int kv) {
  const float inv = fp8_inverse(s), most = s < 247u ? 256.0f : 240.0f;
  auto scaled = [&](uint32_t bits) {
    return __builtin_amdgcn_fmed3f(__uint_as_float(bits) * inv, -most, most);
  };
  const uint32_t c = moe::e4m3_pack4(scaled(a << 16), scaled(a & 0xFFFF0000u), scaled(b << 16),
                                     scaled(b & 0xFFFF0000u));
  return s != kFp8BadScale ? c : kv ? 0u : kFp8NanCodes;
}

// The larger of x over the four lanes of a quad.
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, false));
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, false));
}

// Eight e4m3 codes times a power of two -> bf16, exact.
__device__ __forceinline__ bf16x8 fp8_to_bf16(uint32_t lo, uint32_t hi, float scale) {
  const moe::bf16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const moe::bf16x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const moe::bf16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const moe::bf16x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  bf16x8 r;
  r[0] = p0[0]; r[1] = p0[1]; r[2] = p1[0]; r[3] = p1[1];
  r[4] = p2[0]; r[5] = p2[1]; r[6] = p3[0]; r[7] = p3[1];
  return r;
}

}  // namespace attn
