// Layout and device helpers of the 16-bit paged KV cache and of the attention of prompts (pages_table.hip,
// pages_decode.hip, packed_attn.hip).
//
// A page holds the keys and values of page_size tokens of one sequence in one layer, [2][kv heads][page_size][128]: the
// rows of a head lie one behind the other, so that a workgroup that reads one kv head reads whole runs of memory.  A
// sequence is a row of page ids and a length; the same page id may stand in several rows (refs counts them).
#pragma once

#include "common.h"

namespace lkv {
namespace pages {

constexpr int kD = 128;
constexpr int kMaxSeqs = 2048;  // rows of a page table, sequences of a packed batch (lengths are staged in LDS)
constexpr float kLog2e = 1.4426950408889634f;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct Pages {
  uint16_t* pool;  // [layers][pages][2][H][1 << lg][128]
  int* table;      // [seqs][width]
  int* lens;       // [seqs]
  int* refs;       // [pages]
  int* taken;      // [seqs]
  int layers, pages, H, lg, seqs, width;
};

__host__ __device__ __forceinline__ int page_size(const Pages& st) { return 1 << st.lg; }
// Numbers of a head's rows in one page, and of a page.
__device__ __forceinline__ int64_t run_numbers(const Pages& st) { return static_cast<int64_t>(kD) << st.lg; }
__device__ __forceinline__ int64_t page_numbers(const Pages& st) { return 2 * st.H * run_numbers(st); }
// A sequence's tokens, and the page that an entry of its row names: inside the table and the pool whatever they hold.
__device__ __forceinline__ int held(const Pages& st, int len) { return min(max(len, 0), st.width << st.lg); }
__device__ __forceinline__ int page_id(const Pages& st, int entry) { return min(max(entry, 0), st.pages - 1); }

__device__ __forceinline__ uint32_t pk2(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(lo), static_cast<_Float16>(hi)});
}
__device__ __forceinline__ uint32_t pk2bf(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(lo), static_cast<__bf16>(hi)});
}
template <int DT>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  if constexpr (DT == LKV_DTYPE_F16)
    return pk2(lo, hi);
  else
    return pk2bf(lo, hi);
}
template <int DT>
__device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
  if constexpr (DT == LKV_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}
template <int DT>
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (DT == LKV_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}
// acc + the two numbers of u (exact products with 1, subnormal ones too): sums of softmax weights as they are multiplied, so
// that what rounding does to a weight that outweighs the others cancels in the quotient.
template <int DT>
__device__ __forceinline__ float add_pair(uint32_t u, float acc) {
  if constexpr (DT == LKV_DTYPE_F16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, u), f16x2{static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)},
                                  acc, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, u),
                                           bf16x2{static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)}, acc, false);
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Values that are no numbers, where a product multiplies one that a column does not see by 0: `fine` has 0 in their place and
// `kind` 1 for +inf, 128 for -inf, 129 (both) for NaN, 0 for numbers.  A product of kinds with ones for what a column sees
// counts both, up to 127 of each, and add_counted() adds them to its sum.
template <int DT>
__host__ __device__ __forceinline__ constexpr uint32_t inf_bits() { return DT == LKV_DTYPE_F16 ? 0x7c00u : 0x7f80u; }
template <int DT>
__host__ __device__ __forceinline__ constexpr uint32_t one_bits() { return DT == LKV_DTYPE_F16 ? 0x3c00u : 0x3f80u; }
template <int DT>
__device__ __forceinline__ void no_numbers(const u32x4& raw, u32x4& fine, u32x4& kind) {
  constexpr uint32_t k128 = DT == LKV_DTYPE_F16 ? 0x5800u : 0x4300u, k129 = DT == LKV_DTYPE_F16 ? 0x5808u : 0x4301u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t f = 0, n = 0;
#pragma unroll
    for (int x = 0; x < 32; x += 16) {
      const uint32_t y = raw[j] >> x & 0xffffu, a = y & 0x7fffu;
      f |= (a >= inf_bits<DT>() ? 0u : y) << x;
      n |= (a < inf_bits<DT>() ? 0u : a > inf_bits<DT>() ? k129 : y >> 15 ? k128 : one_bits<DT>()) << x;
    }
    fine[j] = f;
    kind[j] = n;
  }
}
__device__ __forceinline__ void add_counted(float count, float& sum) {
  const float minus = floorf(count * (1.f / 128.f)), plus = count - 128.f * minus;
  if (plus > 0.f) sum += INFINITY;
  if (minus > 0.f) sum -= INFINITY;
}

// log2 of the softmax weights as 16 bits hold them: a new offset puts the largest at 2^top, and there is none until a weight
// passes 2^most, so that most tiles need no rescaled sums.  fp16 keeps a weight's 11 bits down to 2^-20 of the largest.  bf16
// has fp32's exponents, and so do its values: with weights of at most 2^-20 the weighted values of a million tokens add up to
// no more than the largest of them, so that finite ones give finite rows, and values down to 2^-97 are multiplied without
// loss (with fp16's offsets values from 5e36 on gave infinities).
template <int DT>
__host__ __device__ __forceinline__ constexpr float top_weight() { return DT == LKV_DTYPE_F16 ? 6.f : -29.f; }
template <int DT>
__host__ __device__ __forceinline__ constexpr float max_weight() { return DT == LKV_DTYPE_F16 ? 15.f : -20.f; }

// A partial sum's (offset, sum): offset -inf is an empty one, which is passed over.  A row of NaN scores has no offset
// (max passes over NaN) but is not empty: it takes 0, so that its NaN reaches the joined row.
__device__ __forceinline__ float2 part_record(float m, float l) { return float2{l != l ? 0.f : m, l}; }

// Joins the partial sums of rows of 128 numbers (pages_decode.hip): part_ml [rows][splits][2], part_o [rows][splits][128],
// row r's result to out + (r / heads) * o_st + (r % heads) * o_sh.  cu (optional): rows of tokens before cu[0] or from
// cu[n] on are skipped.  So is a row whose first sum is negative.
int launch_join(const float* part_o, const float* part_ml, int64_t rows, int64_t splits, int64_t heads, void* out,
                int64_t o_st, int64_t o_sh, int dtype, const int* cu, int n, hipStream_t stream, const char* what);

// lkv_pages_prefill_attn of a few rows a sequence (pages_decode.hip): up to 32 columns of a kv head, and right for more.
size_t few_rows_bytes(int64_t rows, int64_t S, int64_t Hq, int64_t Hkv, int64_t max_len);
int launch_few_rows(const lkv_pages* p, int64_t layer, const void* q, const int64_t* q_strides, int64_t rows, int64_t Hq,
                    const int32_t* cu, int64_t max_len, float scale, void* out, const int64_t* out_strides, int fill,
                    void* workspace, size_t workspace_bytes, hipStream_t s, const char* what);

// Checks of what the C entries take (pages_table.hip).
int check_pages(const lkv_pages* p, const char* what);
Pages device_pages(const lkv_pages* p);
int check_rows(const void* x, const int64_t* strides, const char* what, const char* name);

}  // namespace pages
}  // namespace lkv
