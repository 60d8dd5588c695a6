// Causal attention of many query rows over the 8-bit block-scaled KV cache (lkv_kv8_attn with more rows per kv head
// than the few-row kernel of kv8_attn.hip takes).
//
// A workgroup of 8 waves owns 256 columns of a kv head, column c the query row (query c / G, head c % G), so that its
// columns end at nearly the same token; a wave has 32.  It walks the blocks of 64 tokens that its columns see.  Each
// block is turned into fp16 numbers (the codes, exactly) in LDS once for all 8 waves: keys [token][dim] by waves 0-3,
// values [dim][token] by waves 4-7, which lie that way in the store already; rows are padded so that 16-byte reads of
// 16 rows fall in distinct banks.  Every wave then runs, on v_mfma_f32_32x32x16_f16,
//   scores^T (32 tokens x 32 columns): A = keys from LDS, B = the wave's queries (registers),
//   softmax: a lane holds 32 of the 64 scores of one column (lane ^ 32 the others),
//   out^T (32 dims x 32 columns) += A = values from LDS, B = the weights from the lane's own registers (the values' token
//   order in LDS is the order in which a lane holds its scores).
// Scales and the running offset are those of kv8_attn.hip; most blocks need no max over lanes and no rescale.
// Two blocks per barrier and two pairs of LDS buffers in turn; waves 4-7 fill the next pair before they compute, waves
// 0-3 after, so that the two waves of a SIMD are out of step.
#include "kv8_common.h"

namespace lkv {
namespace kv8 {
namespace {

constexpr int kWaves = 8;
constexpr int kThr = 64 * kWaves;
constexpr int kCols = 32 * kWaves;
constexpr int kKRow = kD + 8;    // fp16 numbers of a staged key row
constexpr int kVRow = kBlk + 8;  // and of a value row
constexpr int kKBuf = kBlk * kKRow, kVBuf = kD * kVRow;
constexpr int kBufs = 4;
constexpr int kXcds = 8;
constexpr float kHeadroom = 4.f;

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(const f16x8& a, const f16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float half_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ uint32_t cvt2(float a, float b) {
  return __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
}

struct PrefillArgs {
  Store st;
  Rows r;
  int tiles;   // column tiles per (sequence, kv head)
  int chunk, splits;
  float* part_o;
  float* part_ml;
};

template <int DT>
__global__ __launch_bounds__(kThr, 1) void prefill_kernel(PrefillArgs P) {
  __shared__ __align__(16) uint16_t sK[kBufs * kKBuf];
  __shared__ __align__(16) uint16_t sV[kBufs * kVBuf];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c32 = lane & 31, hf = lane >> 5;
  const Store& st = P.st;
  const Rows& r = P.r;
  // Workgroups go to the XCDs round-robin by linear id, and the tiles of one (sequence, kv head) read the same blocks:
  // the items are placed XCD by XCD where their number allows it, the latest queries (the longest) first.
  int tile, split, h, b;
  {
    const int per = P.tiles * P.splits;  // workgroups of an item
    const int items = static_cast<int>(gridDim.x) / per;
    const int p = static_cast<int>(blockIdx.x);
    int item, t;
    if (items % kXcds == 0) {
      const int k = items / kXcds, s = p / kXcds;
      item = p % kXcds + kXcds * (s % k);
      t = s / k;
    } else if (kXcds % items == 0 && per % (kXcds / items) == 0) {
      const int k = kXcds / items, x = p % kXcds;
      item = x % items;
      t = (p / kXcds) * k + x / items;
    } else {
      item = p / per;
      t = p % per;
    }
    // (divisions leave them in vector registers: made scalar again)
    tile = __builtin_amdgcn_readfirstlane(P.tiles - 1 - t / P.splits);
    split = __builtin_amdgcn_readfirstlane(t % P.splits);
    h = __builtin_amdgcn_readfirstlane(item % st.Hkv);
    b = __builtin_amdgcn_readfirstlane(item / st.Hkv);
  }
  const int len = min(max(r.lens[b], 0), r.max_len);
  const int qlen = min(r.q_lens ? min(max(r.q_lens[b], 0), r.S) : r.S, len);
  const int nfull = len / kBlk;
  const int64_t bh = static_cast<int64_t>(b) * st.Hkv + h;
  const int col0 = tile * kCols;
  // ---- the lane's column
  const int col = col0 + 32 * wave + c32, qs = col / r.G, qh = col - qs * r.G;
  const bool ok = col < r.cols && qs < qlen;
  const int lim = ok ? len - qlen + qs + 1 : 0x7fffffff;  // tokens it sees
  f16x8 qf[8];  // B: the column's row, dims 16 kb + 8 hf ..
#pragma unroll
  for (int kb = 0; kb < 8; ++kb) {
    qf[kb] = f16x8{};
    if (ok)
      qf[kb] = load_q8<DT>(r.q, b * r.q_sb + static_cast<int64_t>(h * r.G + qh) * r.q_sh + qs * r.q_ss + 16 * kb + 8 * hf);
  }
  // blocks [blk0, blk1): what the workgroup's last column sees, of the split's
  const int last = min((col0 + kCols - 1) / r.G, qlen - 1);  // its last query
  const int kend = last >= col0 / r.G ? len - qlen + last + 1 : 0;
  const int blk0 = split * P.chunk;
  const int blk1 = min(blk0 + P.chunk, (kend + kBlk - 1) / kBlk);
  // tokens that every column of the wave sees
  const int wq = (col0 + 32 * wave) / r.G;
  const int lim_min = wq < qlen ? len - qlen + wq + 1 : 0x7fffffff;

  // ---- staging: waves 0-3: keys, token kk, dims 32 part ..; waves 4-7: values, dim vd, its tokens of half vh
  const bool key_thr = wave < 4;
  const int kk = (tid & 255) >> 2, part = tid & 3;
  const int vd = (tid & 255) >> 1, vh = tid & 1;
  const uint8_t* const src = (key_thr ? st.k_codes + kk * kD + 32 * part : st.v_codes + vd * kBlk + 16 * vh) +
                             bh * st.blocks * kBlkBytes;
  const int src2 = key_thr ? 16 : 32;  // the thread's second 16 bytes
  uint16_t* const dst = key_thr ? sK + kk * kKRow + 32 * part : sV + vd * kVRow + 8 * vh;
  u32x4 w[2][2];
  auto load_tile = [&](int blk, int u) {
    if (blk < min(blk1, nfull)) {  // uniform
      const uint8_t* p = src + static_cast<int64_t>(blk) * kBlkBytes;
      w[u][0] = *reinterpret_cast<const u32x4*>(p);
      w[u][1] = *reinterpret_cast<const u32x4*>(p + src2);
    }
  };
  auto stage_tile = [&](int blk, int u) {
    const int buf = (blk - blk0) % kBufs;
    uint16_t* d = dst + buf * (key_thr ? kKBuf : kVBuf);
    if (blk < nfull) {
      if (key_thr) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<f16x8*>(d + 8 * k) = codes8h(w[u][k >> 1][2 * (k & 1)], w[u][k >> 1][2 * (k & 1) + 1]);
      } else {
        // step ks of the value product: tokens 16 ks + 4 vh + i, then 16 ks + 8 + 4 vh + i
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) *reinterpret_cast<f16x8*>(d + 16 * ks) = codes8h(w[u][0][ks], w[u][1][ks]);
      }
    } else if (key_thr) {  // the unfinished block: fp16 as it is
      const uint16_t* p = st.k_tail + bh * kBlkBytes + kk * kD + 32 * part;
#pragma unroll
      for (int k = 0; k < 4; ++k) *reinterpret_cast<u32x4*>(d + 8 * k) = *reinterpret_cast<const u32x4*>(p + 8 * k);
    } else {
      const uint16_t* p = st.v_tail + bh * kBlkBytes + vd * kBlk + 16 * vh;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const uint2 a = *reinterpret_cast<const uint2*>(p + 4 * ks), c = *reinterpret_cast<const uint2*>(p + 32 + 4 * ks);
        *reinterpret_cast<u32x4*>(d + 16 * ks) = u32x4{a.x, a.y, c.x, c.y};
      }
    }
  };

  float m = ok ? -INFINITY : 0.f, l = 0.f;  // a column that is no row keeps offset 0 over zero scores
  f32x16 o[4];  // dims 32 db + 8 (i / 4) + 4 hf + i % 4
#pragma unroll
  for (int db = 0; db < 4; ++db) o[db] = f32x16{};

  auto compute_tile = [&](int blk) {
    const int buf = (blk - blk0) % kBufs, t0 = blk * kBlk;
    const uint16_t* k = sK + buf * kKBuf + c32 * kKRow + 8 * hf;
    const uint16_t* v = sV + buf * kVBuf + c32 * kVRow + 8 * hf;
    float kc = r.scale_log2, lv = 0.f, iv = 1.f;
    if (blk < nfull) {  // uniform
      const float2 sc = *reinterpret_cast<const float2*>(st.scales + 2 * (bh * st.blocks + blk));
      const float vs = fmaxf(sc.y, kMinScale);
      kc *= sc.x;
      lv = __log2f(vs);
      iv = __builtin_amdgcn_rcpf(vs);
    }
    f32x16 sc[2];  // token 32 kt + 8 (i / 4) + 4 hf + i % 4
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      sc[kt] = f32x16{};
#pragma unroll
      for (int kb = 0; kb < 8; ++kb)
        sc[kt] = mfma32(*reinterpret_cast<const f16x8*>(k + 32 * kt * kKRow + 16 * kb), qf[kb], sc[kt]);
    }
    float s[32];
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      s[e] = fmaf(sc[e >> 4][e & 15], kc, lv - m);
      mx = fmaxf(mx, s[e]);
    }
    if (t0 + kBlk > lim_min || wave_ballot(mx > 0.f) != 0) {  // uniform
      const int left = lim - t0 - 4 * hf;
      mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float x = fmaf(sc[e >> 4][e & 15], kc, lv);
        s[e] = 8 * (e >> 2) + (e & 3) < left ? x : -INFINITY;
        mx = fmaxf(mx, s[e]);
      }
      mx = half_max(mx);
      const float mn = mx > m ? mx + kHeadroom : m;
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float alpha = exp2_(m - mu);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < 4; ++db) o[db] = o[db] * alpha;
#pragma unroll
      for (int e = 0; e < 32; ++e) s[e] -= mu;
    }
    float ps[2] = {0.f, 0.f};
    f16x8 pf[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      u32x4 u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = exp2_(s[8 * ks + 2 * j]), c = exp2_(s[8 * ks + 2 * j + 1]);
        ps[0] += a;
        ps[1] += c;
        u[j] = cvt2(a, c);
      }
      pf[ks] = __builtin_bit_cast(f16x8, u);
    }
    l = fmaf(ps[0] + ps[1], iv, l);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int db = 0; db < 4; ++db)
        o[db] = mfma32(*reinterpret_cast<const f16x8*>(v + 32 * db * kVRow + 16 * ks), pf[ks], o[db]);
  };

  const int n = max(blk1 - blk0, 0), npair = (n + 1) / 2;
  auto next_pair = [&](int it) {
    const int blk = blk0 + 2 * it;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (blk + u < blk1) stage_tile(blk + u, u);
#pragma unroll
    for (int u = 0; u < 2; ++u) load_tile(blk + 2 + u, u);
  };
  if (npair) {
    load_tile(blk0, 0);
    load_tile(blk0 + 1, 1);
    next_pair(0);
  }
  __syncthreads();
#pragma unroll 1
  for (int it = 0; it < npair; ++it) {
    if (!key_thr && it + 1 < npair) next_pair(it + 1);
#pragma unroll 1
    for (int blk = blk0 + 2 * it; blk < min(blk0 + 2 * it + 2, blk1); ++blk) compute_tile(blk);
    if (key_thr && it + 1 < npair) next_pair(it + 1);
    __syncthreads();
  }

  if (col >= r.cols) return;
  l = half_sum(l);
  if (P.splits == 1) {
    const bool some = ok && l != 0.f;
    const float inv = some ? 1.f / l : 0.f;
    const int64_t at = b * r.o_sb + static_cast<int64_t>(h * r.G + qh) * r.o_sh + qs * r.o_ss + 4 * hf;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = some ? o[db][4 * k + i] * inv : 0.f;
        store4<DT>(r.out, at + 32 * db + 8 * k, x[0], x[1], x[2], x[3]);
      }
  } else {
    const int64_t at = (bh * r.cols + col) * P.splits + split;
    const bool some = ok && n > 0;
    if (hf == 0) *reinterpret_cast<float2*>(P.part_ml + 2 * at) = some ? float2{m, l} : float2{-INFINITY, 0.f};
    if (some) {
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<f32x4*>(P.part_o + at * kD + 32 * db + 8 * k + 4 * hf) =
              f32x4{o[db][4 * k], o[db][4 * k + 1], o[db][4 * k + 2], o[db][4 * k + 3]};
    }
  }
}

}  // namespace

int launch_prefill(const Store& store, const Rows& r, const Plan& p, int dtype, int64_t B, float* part_o,
                   float* part_ml, hipStream_t stream) {
  const PrefillArgs A{store, r, p.groups, p.chunk, p.splits, part_o, part_ml};
  const int64_t wgs = B * store.Hkv * p.groups * p.splits;
  LKV_REQUIRE(wgs < (1ll << 31), "kv8_attn: %lld workgroups", (long long)wgs);
  const dim3 grid(static_cast<unsigned>(wgs));
  if (dtype == LKV_DTYPE_F32)
    hipLaunchKernelGGL(prefill_kernel<LKV_DTYPE_F32>, grid, dim3(kThr), 0, stream, A);
  else if (dtype == LKV_DTYPE_F16)
    hipLaunchKernelGGL(prefill_kernel<LKV_DTYPE_F16>, grid, dim3(kThr), 0, stream, A);
  else
    hipLaunchKernelGGL(prefill_kernel<LKV_DTYPE_BF16>, grid, dim3(kThr), 0, stream, A);
  LKV_LAUNCH_CHECK("kv8_attn prefill");
  return LKV_OK;
}

}  // namespace kv8
}  // namespace lkv
