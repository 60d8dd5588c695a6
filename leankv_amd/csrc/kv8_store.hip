// 8-bit block-scaled KV cache: storing tokens and reading them back (layout in kv8_common.h).
//
// lkv_kv8_update, one launch, one workgroup of 256 threads for each (key or value, sequence, kv head, touched block).
// A block that the new tokens finish is quantized from the unfinished block's fp16 tokens and the new ones: its 64 x 128
// values lie in registers (a thread has 8 dims of 4 consecutive tokens, read in 16-byte rows), one max over the
// workgroup gives the scale, and the codes go out in 8-byte pieces (keys) or through LDS as [dim][position] rows
// (values: the 4 tokens of a thread's dim are one dword of the row, so the transpose is dword moves).  Tokens that
// finish no block go to the fp16 tail.  The workgroup of the first touched block also writes the new tail, after its
// own reads of the old one, so no other workgroup touches the tail.
// Bound by memory for prompts: a value is read once (2 bytes) and written once (1 byte); 8 x 4096 tokens of 8 heads, 201 MB,
// 49 us in a replayed graph over six stores in turn (4.1 TB/s; a device copy 5.0), 37 over one store, which stays in the
// last-level cache.  Sixteen ragged prompts of up to 1201 tokens 31 us traced (2.3 TB/s): the grid is for the longest, over
// 40 % of the workgroups find no block.  4096 tokens of one sequence 10.3 us (40 stores in turn), one token 2.8 us, or 4.5
// where it finishes a block (an empty launch 2.1).  What a value costs in instructions matters as much: magnitudes are
// compared as bits, two at a time, and a code is one product and one addition (10.1 -> 9.1 us for 4096 tokens, profiled).
#include "kv8_common.h"

namespace lkv {
namespace kv8 {
namespace {

constexpr int kThr = 256;
constexpr int kVRow = 17;  // dwords of a staged value row: 16 and one of padding

__device__ __forceinline__ uint32_t xg_min(uint32_t v) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  auto mn = [](uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(s16x2, a), __builtin_bit_cast(s16x2, b)));
  };
  auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = mn(a[0], a[1]);
  a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return mn(a[0], a[1]);
}

struct UpdateArgs {
  Store st;
  const void* x[2];           // keys, values
  int64_t sb[2], sh[2], ss[2];  // strides in elements
  const int* pos;             // [B] tokens held before
  const int* n_new;           // [B] or null
  int S;
};

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t umax2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ float half_lo(uint32_t u) { return static_cast<float>(__builtin_bit_cast(f16x2, u)[0]); }
__device__ __forceinline__ float half_hi(uint32_t u) { return static_cast<float>(__builtin_bit_cast(f16x2, u)[1]); }

// Eight numbers as stored, in fp16 pairs.  A row holds an infinity, a NaN or a number past fp16 now and then only: the
// largest magnitude (as bits, two at a time) tells, and only then is every number looked at.
template <int DT>
__device__ __forceinline__ u32x4 load_kv8(const void* base, int64_t at) {
  if constexpr (DT == LKV_DTYPE_F32) {
    float x[8];
    load8<DT>(base, at, x);
    u32x4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = pk2(clamp_kv(x[2 * j]), clamp_kv(x[2 * j + 1]));
    return r;
  } else {
    u32x4 u = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(base) + at);
    constexpr uint32_t kAbs = 0x7fff7fffu;
    const uint32_t m = umax2(umax2(u[0] & kAbs, u[1] & kAbs), umax2(u[2] & kAbs, u[3] & kAbs));
    constexpr uint32_t kFirst = DT == LKV_DTYPE_F16 ? 0x7c00u : 0x4780u;  // infinity; 65536 in bf16
    const bool special = max(m & 0xffffu, m >> 16) >= kFirst;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b;
      if constexpr (DT == LKV_DTYPE_F16)
        a = half_lo(u[j]), b = half_hi(u[j]);
      else
        a = bf2f(u[j] & 0xffffu), b = __uint_as_float(u[j] & 0xffff0000u);
      if (special) a = clamp_kv(a), b = clamp_kv(b);
      if (DT != LKV_DTYPE_F16 || special) u[j] = pk2(a, b);
    }
    return u;
  }
}

// thread: dims 8 c .. 8 c + 7 of tokens 4 a .. 4 a + 3 of the block
template <int DT>
__global__ __launch_bounds__(kThr) void update_kernel(UpdateArgs P) {
  __shared__ uint32_t s_max[4];
  __shared__ uint32_t s_rng[4][2][64];
  __shared__ uint32_t s_v[kD * kVRow];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = tid & 15, a = tid >> 4;
  const int which = blockIdx.y & 1;  // 0 keys, 1 values
  const int h = blockIdx.y >> 1, b = blockIdx.z;
  const Store& st = P.st;
  // the sequence's tokens [p0, p1); a position outside the store stores nothing, tokens past it are dropped
  const int64_t cap = static_cast<int64_t>(st.blocks) * kBlk;
  const int64_t p0 = P.pos[b];
  const int64_t n = min(static_cast<int64_t>(P.n_new ? P.n_new[b] : P.S), static_cast<int64_t>(P.S));
  if (p0 < 0 || p0 >= cap || n <= 0) return;
  const int64_t p1 = min(p0 + n, cap);
  const int64_t blk = p0 / kBlk + blockIdx.x;
  const int64_t t0 = blk * kBlk;  // first token of this block
  if (t0 >= p1) return;
  const bool first = blockIdx.x == 0;
  const bool done = t0 + kBlk <= p1;
  if (!done && !first) return;  // the unfinished block is the first workgroup's

  const int64_t bh = static_cast<int64_t>(b) * st.Hkv + h;
  const void* x = P.x[which];
  const int64_t xrow = b * P.sb[which] + h * P.sh[which] + 8 * c;
  auto tail_of = [&](int64_t j) { return tail_ptr(st, which, bh, j); };
  // the unfinished block behind the new tokens, and whether the last finished one shares the tail that the first
  // workgroup reads
  const int64_t open = p1 / kBlk, before = p0 / kBlk;
  const bool shared = open - 1 > before && !((open - 1 - before) & 1) && p0 % kBlk;

  if (done) {
    u32x4 v[4];  // token 4 a + i: fp16 pairs of its 8 dims
    // older tokens of the block: those before p0 (none but in the first block)
    const int old = first ? static_cast<int>(p0 - t0) : 0;
    uint16_t* const tail = tail_of(blk);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 4 * a + i;
      if (t >= old)
        v[i] = load_kv8<DT>(x, xrow + (t0 + t - p0) * P.ss[which]);
      else if (!which)
        v[i] = *reinterpret_cast<const u32x4*>(tail + t * kD + 8 * c);
    }
    if (which && 4 * a < old) {
      uint2 vt[8];  // four tokens of a dim
#pragma unroll
      for (int j = 0; j < 8; ++j) vt[j] = *reinterpret_cast<const uint2*>(tail + (8 * c + j) * kBlk + 4 * v_dword(a));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * a + i < old) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t lo = i < 2 ? vt[2 * j].x : vt[2 * j].y, hi = i < 2 ? vt[2 * j + 1].x : vt[2 * j + 1].y;
            v[i][j] = __builtin_amdgcn_perm(hi, lo, (i & 1) ? 0x07060302u : 0x05040100u);
          }
        }
    }
    // the largest magnitude, as bits (all are finite)
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) m = umax2(m, v[i][j] & 0x7fff7fffu);
    m = max(m & 0xffffu, m >> 16);
    const uint32_t wm = __float_as_uint(wave_max(h2f(static_cast<uint16_t>(m))));
    if (lane == 0) s_max[wave] = wm;
    __syncthreads();
    const float amax = fmaxf(fmaxf(__uint_as_float(s_max[0]), __uint_as_float(s_max[1])),
                             fmaxf(__uint_as_float(s_max[2]), __uint_as_float(s_max[3])));
    const float inv = code_factor(amax);
    // codes in units: the product rounded, then rounded to a whole number by adding 1.5 * 2^23 (+ 128): the sum's low
    // byte is code + 128; |x * inv| <= 127 (1 + 2^-22) rounds to 127 at most
    constexpr float kMagic = 12582912.f + 128.f;
    float t[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t[i][2 * j] = fmaf(half_lo(v[i][j]), inv, 0.f);
        t[i][2 * j + 1] = fmaf(half_hi(v[i][j]), inv, 0.f);
      }
    auto bytes = [](float a0, float a1, float a2, float a3) {
      const uint32_t u0 = __float_as_uint(a0 + kMagic), u1 = __float_as_uint(a1 + kMagic),
                     u2 = __float_as_uint(a2 + kMagic), u3 = __float_as_uint(a3 + kMagic);
      return __builtin_amdgcn_perm(__builtin_amdgcn_perm(u3, u2, 0x0c0c0400u), __builtin_amdgcn_perm(u1, u0, 0x0c0c0400u),
                                   0x05040100u);
    };
    const int64_t at = bh * st.blocks + blk;
    if (tid == 0) st.scales[2 * at + which] = amax * kStep;
    if (!which) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint2*>(st.k_codes + at * kBlkBytes + (4 * a + i) * kD + 8 * c) =
            uint2{bytes(t[i][0], t[i][1], t[i][2], t[i][3]), bytes(t[i][4], t[i][5], t[i][6], t[i][7])};
      // lowest and highest code of every dim, two dims in a dword: over the thread's 4 tokens, the wave's 16, the block's
      // 64 (the highest as the negated lowest of the negated codes)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t lo[2], hi[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int d = 2 * j + k;
          lo[k] = __float_as_uint(fminf(fminf(t[0][d], t[1][d]), fminf(t[2][d], t[3][d])) + 12582912.f);
          hi[k] = __float_as_uint(12582912.f - fmaxf(fmaxf(t[0][d], t[1][d]), fmaxf(t[2][d], t[3][d])));
        }
        const uint32_t l2 = xg_min(__builtin_amdgcn_perm(lo[1], lo[0], 0x05040100u));
        const uint32_t h2 = xg_min(__builtin_amdgcn_perm(hi[1], hi[0], 0x05040100u));
        if (lane < 16) {
          s_rng[wave][0][4 * c + j] = l2;
          s_rng[wave][1][4 * c + j] = h2;
        }
      }
      __syncthreads();
      // dims 2 d2, 2 d2 + 1
      if (tid < 128) {
        const int d2 = tid & 63, hi = tid >> 6;
        int r0 = 127, r1 = 127;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t u = s_rng[w][hi][d2];
          r0 = min(r0, static_cast<int>(static_cast<int16_t>(u & 0xffffu)));
          r1 = min(r1, static_cast<int>(static_cast<int16_t>(u >> 16)));
        }
        if (hi) r0 = -r0, r1 = -r1;
        reinterpret_cast<uint16_t*>(st.ranges + at * 2 * kD + hi * kD)[d2] =
            static_cast<uint16_t>((r0 & 0xff) | ((r1 & 0xff) << 8));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) s_v[(8 * c + j) * kVRow + v_dword(a)] = bytes(t[0][j], t[1][j], t[2][j], t[3][j]);
      __syncthreads();
      // two 16-byte pieces a thread
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int piece = k * kThr + tid, d = piece >> 2, q = 4 * (piece & 3);
        const uint32_t* s = s_v + d * kVRow + q;
        *reinterpret_cast<u32x4*>(st.v_codes + at * kBlkBytes + d * kBlk + 4 * q) = u32x4{s[0], s[1], s[2], s[3]};
      }
    }
    // the last finished block's new tokens, as they are.  From the registers and behind the barriers, which wait for
    // stores: a token that finishes a block of 64 sequences, with its read-back, 16.1 us (before them 16.6, not kept at
    // all 15.1); read again 16.2, and 4096 tokens 18.5 instead of 15.1.
    if (blk == open - 1 && !shared) {
      if (!which) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * a + i >= old) *reinterpret_cast<u32x4*>(tail + (4 * a + i) * kD + 8 * c) = v[i];
      } else if (4 * a + 3 >= old) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // the four tokens of a dim (older ones among them as they were)
          const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
          *reinterpret_cast<uint2*>(tail + (8 * c + j) * kBlk + 4 * v_dword(a)) =
              uint2{__builtin_amdgcn_perm(v[1][j >> 1], v[0][j >> 1], sel),
                    __builtin_amdgcn_perm(v[3][j >> 1], v[2][j >> 1], sel)};
        }
      }
    }
  }
  if (!first) return;
  // the new tokens of the unfinished block, and of the last finished one where its own workgroup left them, in their slots
  __syncthreads();  // (every read of older tokens is done)
  if (tid == 0 && p1 > open * kBlk) st.scales[2 * (bh * st.blocks + open) + which] = kOpenScale;
#pragma unroll 1
  for (int64_t j = shared ? open - 1 : open; j <= open; ++j) {
    uint16_t* const tail = tail_of(j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int slot = 4 * a + i;
      const int64_t t = j * kBlk + slot;
      if (t < p0 || t >= p1) continue;
      const u32x4 y = load_kv8<DT>(x, xrow + (t - p0) * P.ss[which]);
      if (!which) {
        *reinterpret_cast<u32x4*>(tail + slot * kD + 8 * c) = y;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          tail[(8 * c + 2 * k) * kBlk + v_pos(slot)] = static_cast<uint16_t>(y[k] & 0xffffu);
          tail[(8 * c + 2 * k + 1) * kBlk + v_pos(slot)] = static_cast<uint16_t>(y[k] >> 16);
        }
      }
    }
  }
}

struct ReadArgs {
  Store st;
  const int* lens;
  uint16_t* out[2];  // keys, values: fp16 [B][Hkv][n][128]
  int64_t first, n;  // tokens first .. first + n - 1
};

// One workgroup per (key or value, sequence, kv head, block of 64 tokens): codes in 16-byte pieces, values through LDS
// back to rows, fp16 rows out in 16-byte pieces.  Bound by memory: 8 x 4096 tokens of 8 heads, 201 MB, 34 us
// (5.9 TB/s, six stores in turn).
__global__ __launch_bounds__(kThr) void read_kernel(ReadArgs P) {
  __shared__ uint32_t s_v[kD * kVRow];
  const int tid = threadIdx.x;
  const int c = tid & 15, a = tid >> 4;
  const int which = blockIdx.y & 1, h = blockIdx.y >> 1, b = blockIdx.z;
  const Store& st = P.st;
  const int64_t cap = static_cast<int64_t>(st.blocks) * kBlk;
  const int64_t len = min(max(static_cast<int64_t>(P.lens[b]), static_cast<int64_t>(0)), cap);
  const int64_t blk = P.first / kBlk + blockIdx.x, t0 = blk * kBlk;
  const int64_t bh = static_cast<int64_t>(b) * st.Hkv + h;
  const bool done = t0 + kBlk <= len;
  const int64_t at = bh * st.blocks + blk;
  uint32_t w[4][4];  // token 4 a + i, dims 8 c .. as fp16 pairs
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) w[i][j] = 0;
  if (done) {
    const float scale = st.scales[2 * at + which];
    // fp16(code * scale), the product in fp32
    auto vals = [&](uint32_t codes) {
      return pk2(fmaf(half_lo(codes), scale, 0.f), fmaf(half_hi(codes), scale, 0.f));
    };
    if (!which) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint2 u = *reinterpret_cast<const uint2*>(st.k_codes + at * kBlkBytes + (4 * a + i) * kD + 8 * c);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i][j] = vals(codes2h(j < 2 ? u.x : u.y, (j & 1) ? kSelHi : kSelLo));
      }
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int piece = k * kThr + tid, d = piece >> 2, q = 4 * (piece & 3);
        const u32x4 u = *reinterpret_cast<const u32x4*>(st.v_codes + at * kBlkBytes + d * kBlk + 4 * q);
#pragma unroll
        for (int j = 0; j < 4; ++j) s_v[d * kVRow + q + j] = u[j];
      }
      __syncthreads();
      uint32_t u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = s_v[(8 * c + j) * kVRow + v_dword(a)];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[i][j] = vals(codes2h(__builtin_amdgcn_perm(u[2 * j + 1], u[2 * j], 0x0c0c0400u + 0x0101u * i), kSelLo));
    }
  } else if (t0 < len) {
    const uint16_t* tail = tail_ptr(st, which, bh, blk);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 4 * a + i;
      if (t0 + t >= len) continue;
      if (!which) {
        const u32x4 u = *reinterpret_cast<const u32x4*>(tail + t * kD + 8 * c);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i][j] = u[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[i][j] = static_cast<uint32_t>(tail[(8 * c + 2 * j) * kBlk + v_pos(t)]) |
                    (static_cast<uint32_t>(tail[(8 * c + 2 * j + 1) * kBlk + v_pos(t)]) << 16);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t t = t0 + 4 * a + i - P.first;
    if (t < 0 || t >= P.n) continue;
    *reinterpret_cast<u32x4*>(P.out[which] + (bh * P.n + t) * kD + 8 * c) = u32x4{w[i][0], w[i][1], w[i][2], w[i][3]};
  }
}

}  // namespace
}  // namespace kv8
}  // namespace lkv

using namespace lkv;
using namespace lkv::kv8;

namespace lkv {
namespace kv8 {

int check_store(const lkv_kv8_store* s, const char* what) {
  LKV_REQUIRE(s, "%s: null store", what);
  LKV_REQUIRE(s->batch >= 0 && s->batch < 65536 && s->kv_heads > 0 && s->kv_heads < 32768 && s->blocks > 0 &&
                  s->blocks < (1ll << 24),
              "%s: store of %lld sequences, %lld kv heads, %lld blocks out of range", what, (long long)s->batch,
              (long long)s->kv_heads, (long long)s->blocks);
  LKV_REQUIRE(s->batch == 0 || (s->k_codes && s->v_codes && s->scales && s->ranges && s->k_tail && s->v_tail),
              "%s: null pointer in the store", what);
  LKV_REQUIRE(aligned16(s->k_codes) && aligned16(s->v_codes) && aligned16(s->scales) && aligned16(s->ranges) &&
                  aligned16(s->k_tail) && aligned16(s->v_tail),
              "%s: the store's buffers must be 16-byte aligned", what);
  return LKV_OK;
}

Store device_store(const lkv_kv8_store* s) {
  Store d;
  d.k_codes = static_cast<uint8_t*>(s->k_codes);
  d.v_codes = static_cast<uint8_t*>(s->v_codes);
  d.scales = static_cast<float*>(s->scales);
  d.ranges = static_cast<int8_t*>(s->ranges);
  d.k_tail = static_cast<uint16_t*>(s->k_tail);
  d.v_tail = static_cast<uint16_t*>(s->v_tail);
  d.Hkv = static_cast<int>(s->kv_heads);
  d.blocks = static_cast<int>(s->blocks);
  return d;
}

int check_rows(const void* x, const int64_t* strides, int dtype, const char* what, const char* name) {
  const int64_t unit = dtype == LKV_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
  LKV_REQUIRE(aligned16(x) && strides && strides[0] % unit == 0 && strides[1] % unit == 0 && strides[2] % unit == 0,
              "%s: rows of %s must be 16-byte aligned", what, name);
  return LKV_OK;
}

}  // namespace kv8
}  // namespace lkv

extern "C" int lkv_kv8_update(const lkv_kv8_store* store, const void* k, const int64_t* k_strides, const void* v,
                              const int64_t* v_strides, int dtype, int64_t S, const int32_t* pos, const int32_t* n_new,
                              void* stream) {
  if (int rc = check_store(store, "kv8_update")) return rc;
  LKV_REQUIRE(dtype == LKV_DTYPE_F32 || dtype == LKV_DTYPE_F16 || dtype == LKV_DTYPE_BF16, "kv8_update: dtype %d", dtype);
  LKV_REQUIRE(S >= 0 && S < (1ll << 30), "kv8_update: S=%lld out of range", (long long)S);
  if (store->batch == 0 || S == 0) return LKV_OK;
  LKV_REQUIRE(k && v && pos, "kv8_update: null pointer");
  if (int rc = check_rows(k, k_strides, dtype, "kv8_update", "k")) return rc;
  if (int rc = check_rows(v, v_strides, dtype, "kv8_update", "v")) return rc;
  UpdateArgs P;
  P.st = device_store(store);
  P.x[0] = k;
  P.x[1] = v;
  for (int w = 0; w < 2; ++w) {
    const int64_t* s = w ? v_strides : k_strides;
    P.sb[w] = s[0];
    P.sh[w] = s[1];
    P.ss[w] = s[2];
  }
  P.pos = pos;
  P.n_new = n_new;
  P.S = static_cast<int>(S);
  // blocks that S tokens from any position touch
  const dim3 grid(static_cast<unsigned>((S + kBlk - 2) / kBlk + 1), static_cast<unsigned>(2 * store->kv_heads),
                  static_cast<unsigned>(store->batch));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == LKV_DTYPE_F32)
    hipLaunchKernelGGL(update_kernel<LKV_DTYPE_F32>, grid, dim3(kThr), 0, st, P);
  else if (dtype == LKV_DTYPE_F16)
    hipLaunchKernelGGL(update_kernel<LKV_DTYPE_F16>, grid, dim3(kThr), 0, st, P);
  else
    hipLaunchKernelGGL(update_kernel<LKV_DTYPE_BF16>, grid, dim3(kThr), 0, st, P);
  LKV_LAUNCH_CHECK("kv8_update");
  return LKV_OK;
}

extern "C" int lkv_kv8_read(const lkv_kv8_store* store, const int32_t* lens, int64_t first, int64_t n, void* k, void* v,
                            void* stream) {
  if (int rc = check_store(store, "kv8_read")) return rc;
  const int64_t cap = store->blocks * kBlk;
  LKV_REQUIRE(first >= 0 && first <= cap && n >= 0 && n <= cap - first,
              "kv8_read: %lld tokens from %lld on outside a store of %lld", (long long)n, (long long)first,
              (long long)cap);
  if (store->batch == 0 || n == 0) return LKV_OK;
  LKV_REQUIRE(lens && k && v, "kv8_read: null pointer");
  LKV_REQUIRE(aligned16(k) && aligned16(v), "kv8_read: outputs must be 16-byte aligned");
  ReadArgs P;
  P.st = device_store(store);
  P.lens = lens;
  P.out[0] = static_cast<uint16_t*>(k);
  P.out[1] = static_cast<uint16_t*>(v);
  P.first = first;
  P.n = n;
  const int64_t nb = (first + n - 1) / kBlk - first / kBlk + 1;
  hipLaunchKernelGGL(read_kernel, dim3(static_cast<unsigned>(nb), static_cast<unsigned>(2 * store->kv_heads),
                                       static_cast<unsigned>(store->batch)),
                     dim3(kThr), 0, static_cast<hipStream_t>(stream), P);
  LKV_LAUNCH_CHECK("kv8_read");
  return LKV_OK;
}
