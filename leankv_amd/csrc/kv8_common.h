// Layout and device helpers of the 8-bit block-scaled KV cache (kv8_store.hip, kv8_attn.hip, kv8_prefill.hip).
//
// A finished block is 64 tokens of one kv head.  Its 64 x 128 keys share one scale, so do its values:
//   scale = amax / 127, code = rint(x * (127 / amax)) in -127 .. 127, value = code * scale
// (in fp32 with the roundings of amax * fp32(1 / 127) and x * (127 * (1 / amax))), and a code is stored as the byte
// code + 128.  Keys lie [token][dim].  Values lie [dim][position], so that the value product reads its operand (8 tokens
// of one dim per lane) as it lies in memory, with no transpose in the attention kernels; position 16 g + 8 ks + 4 t + i
// holds token 32 ks + 16 t + 4 g + i: the tokens whose weights lane group g of a wave has after the 16-row score products
// 2 ks and 2 ks + 1.  The unfinished block of a head is fp16 in the same two layouts.  So is, next to its codes, the last
// finished one, so that a sequence can be taken back into it: block j's fp16 tokens lie in tail j & 1.
#pragma once

#include "common.h"

namespace lkv {
namespace kv8 {

constexpr int kD = 128;
constexpr int kBlk = 64;
constexpr int kBlkBytes = kBlk * kD;  // codes of one block of keys (or values)
constexpr float kF16Max = 65504.f;
constexpr float kLog2e = 1.4426950408889634f;
// Values of a block enter the softmax weights as a power of two (see kv8_attn.hip); a block of zeros takes this one.
constexpr float kMinScale = 4.656612873077393e-10f;  // 2^-31, below 2^-24 / 127, the smallest scale of a nonzero block

// log2 of the softmax weights as fp16 holds them: a new offset puts the largest at 2^6, and there is none until a weight
// passes 2^15, so that most blocks need no max over lanes and no rescaled sums.  A weight keeps fp16's 11 bits down to
// 2^-20 of the largest.
constexpr float kTopWeight = 6.f, kMaxWeight = 15.f;

constexpr float kStep = 1.f / 127.f;
// What numbers with the largest magnitude amax are multiplied by before they are rounded to codes.
__device__ __forceinline__ float code_factor(float amax) { return amax > 0.f ? (1.f / amax) * 127.f : 0.f; }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct Store {
  uint8_t* k_codes;   // [B][Hkv][blocks][64][128]
  uint8_t* v_codes;   // [B][Hkv][blocks][128][64]
  float* scales;      // [B][Hkv][blocks][2]: key, value
  int8_t* ranges;     // [B][Hkv][blocks][2][128]: lowest and highest key code of a dim
  uint16_t* k_tail;   // fp16 [B][Hkv][2][64][128]
  uint16_t* v_tail;   // fp16 [B][Hkv][2][128][64]
  int Hkv, blocks;
};

// Block j's fp16 tokens of (sequence, kv head) bh.
__device__ __forceinline__ uint16_t* tail_ptr(const Store& st, bool values, int64_t bh, int64_t j) {
  return (values ? st.v_tail : st.k_tail) + (2 * bh + (j & 1)) * kBlkBytes;
}
constexpr float kOpenScale = -1.f;  // in the scales' place of an unfinished block

// Value position of the dword of tokens 4 a .. 4 a + 3 (a = 8 ks + 4 t + g -> 4 g + 2 ks + t).
__host__ __device__ __forceinline__ constexpr int v_dword(int a) { return 4 * (a & 3) + (a >> 2); }
// Value position of token t of its block.
__host__ __device__ __forceinline__ constexpr int v_pos(int t) { return 4 * v_dword(t >> 2) + (t & 3); }
static_assert(v_pos(0) == 0 && v_pos(4) == 16 && v_pos(16) == 4 && v_pos(32) == 8 && v_pos(63) == 63, "value order");

__device__ __forceinline__ uint32_t pk2(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(lo), static_cast<_Float16>(hi)});
}
__device__ __forceinline__ float bf2f(uint32_t h) { return __uint_as_float(h << 16); }

// Two stored codes (bytes of w picked by a selector) as the fp16 numbers code, exact: a byte u under the fp16
// exponent of 1024 is 1024 + u, and 1024 + 128 comes off.
constexpr uint32_t kSelLo = 0x04010400u, kSelHi = 0x04030402u;
__device__ __forceinline__ uint32_t codes2h(uint32_t w, uint32_t sel) {
  const f16x2 v = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, sel)) -
                  f16x2{static_cast<_Float16>(1152.f), static_cast<_Float16>(1152.f)};
  return __builtin_bit_cast(uint32_t, v);
}
// Eight codes (two dwords) as an MFMA operand.
__device__ __forceinline__ f16x8 codes8h(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(f16x8, u32x4{codes2h(a, kSelLo), codes2h(a, kSelHi), codes2h(b, kSelLo), codes2h(b, kSelHi)});
}

// Eight consecutive elements of type DT (LKV_DTYPE_*) from a 16-byte aligned address, as fp32.
template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&x)[8]) {
  if constexpr (DT == LKV_DTYPE_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    const float4 a = p[0], b = p[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const u32x4 u = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(base) + at);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == LKV_DTYPE_F16) {
        x[2 * j] = h2f(static_cast<uint16_t>(u[j] & 0xffffu));
        x[2 * j + 1] = h2f(static_cast<uint16_t>(u[j] >> 16));
      } else {
        x[2 * j] = bf2f(u[j] & 0xffffu);
        x[2 * j + 1] = bf2f(u[j] >> 16);
      }
    }
  }
}
// Queries as the kernels multiply them: fp16, infinities and larger numbers at the largest one, a NaN stays.
__device__ __forceinline__ float clamp_q(float x) {
  const float c = fminf(fmaxf(x, -kF16Max), kF16Max);
  return x != x ? x : c;
}
// Keys and values as they are stored: the same, but a NaN is a 0 (one would make its whole block NaN).
__device__ __forceinline__ float clamp_kv(float x) {
  const float c = fminf(fmaxf(x, -kF16Max), kF16Max);
  return x != x ? 0.f : c;
}
// The same for two fp16 numbers: an infinity (0x7c00 without its sign) becomes the number before it.
__device__ __forceinline__ uint32_t clamp_q2(uint32_t u) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  const u16x2 x = __builtin_bit_cast(u16x2, u), one = u16x2{1, 1};
  const u16x2 t = (x & u16x2{0x7fff, 0x7fff}) - u16x2{0x7c00, 0x7c00};
  return __builtin_bit_cast(uint32_t, static_cast<u16x2>(x + (__builtin_elementwise_min(t, one) - one)));
}
// Eight elements of a query row as they lie in memory, and as fp16.
template <int DT>
struct RawQ {
  u32x4 u[DT == LKV_DTYPE_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ RawQ<DT> load_raw_q8(const void* base, int64_t at) {
  RawQ<DT> r;
  const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const char*>(base) + at * (DT == LKV_DTYPE_F32 ? 4 : 2));
#pragma unroll
  for (int k = 0; k < (DT == LKV_DTYPE_F32 ? 2 : 1); ++k) r.u[k] = p[k];
  return r;
}
template <int DT>
__device__ __forceinline__ f16x8 convert_q8(const RawQ<DT>& q) {
  u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (DT == LKV_DTYPE_F16)
      r[j] = clamp_q2(q.u[0][j]);
    else if constexpr (DT == LKV_DTYPE_BF16)
      r[j] = pk2(clamp_q(bf2f(q.u[0][j] & 0xffffu)), clamp_q(bf2f(q.u[0][j] >> 16)));
    else
      r[j] = pk2(clamp_q(__uint_as_float(q.u[j >> 1][2 * (j & 1)])), clamp_q(__uint_as_float(q.u[j >> 1][2 * (j & 1) + 1])));
  }
  return __builtin_bit_cast(f16x8, r);
}
template <int DT>
__device__ __forceinline__ f16x8 load_q8(const void* base, int64_t at) {
  return convert_q8<DT>(load_raw_q8<DT>(base, at));
}

// Four consecutive outputs of type DT at element offset `at` (a multiple of 4; the row is 16-byte aligned).
__device__ __forceinline__ uint32_t pk2bf(float lo, float hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(lo), static_cast<__bf16>(hi)});
}
template <int DT>
__device__ __forceinline__ void store4(void* base, int64_t at, float a, float b, float c, float d) {
  if constexpr (DT == LKV_DTYPE_F32)
    *reinterpret_cast<float4*>(static_cast<float*>(base) + at) = float4{a, b, c, d};
  else if constexpr (DT == LKV_DTYPE_F16)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) = uint2{pk2(a, b), pk2(c, d)};
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) = uint2{pk2bf(a, b), pk2bf(c, d)};
}

// Max / sum over the four lanes of a wave that share lane % 16 (one softmax column).
__device__ __forceinline__ float groups_max(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// A partial sum's (offset, sum): offset -inf is an empty one, which is passed over.  A row of NaN scores has no offset
// (max passes over NaN) but is not empty: it takes 0, so that its NaN reaches the joined row.
__device__ __forceinline__ float2 part_record(float m, float l) { return float2{l != l ? 0.f : m, l}; }

// A sequence's tokens: its length; one that is longer than the caller's bound ends with the last finished block below it (its
// queries' positions count from that end too).
__device__ __forceinline__ int held_tokens(int len, int max_len) {
  return len > max_len ? max_len & ~(kBlk - 1) : max(len, 0);
}

// Query rows of one kv head as the columns of its score products: column c is query c / G, head c % G.
struct Rows {
  const void* q;
  int64_t q_sb, q_sh, q_ss;  // strides in elements
  void* out;
  int64_t o_sb, o_sh, o_ss;
  const int* lens;    // [B] tokens held, the queries' own among them
  const int* q_lens;  // [B] queries of a sequence, or null: all S
  int G, S, cols;     // cols = S * G
  int max_len;        // bound on lens
  float scale_log2;   // scale * log2(e)
};

// What a launch does, from the shapes alone (never from what the device tensors hold).
struct Plan {
  int nt;       // 16-column tiles per block of the few-row kernel, 0: the many-row kernel
  int groups;   // column groups per (sequence, kv head)
  int chunk;    // key blocks per split
  int splits;
};
Plan make_plan(int64_t B, int64_t Hkv, int64_t cols, int64_t units, bool listed);
size_t plan_bytes(const Plan& p, int64_t B, int64_t Hkv, int64_t cols);
int launch_prefill(const Store& st, const Rows& r, const Plan& p, int dtype, int64_t B, float* part_o, float* part_ml,
                   hipStream_t stream);

}  // namespace kv8
}  // namespace lkv
