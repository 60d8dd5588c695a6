// Attention of few query rows over the 8-bit block-scaled KV cache, and the choice of blocks for sparse attention.
//
// Decode attention (lkv_kv8_attn with few rows): one launch over the cache, one that joins the splits.
//   split kernel  grid (splits, kv heads x column groups, sequences), 4 waves.  The columns of a kv head are its query
//                 rows (query, head).  A wave takes every 4th block of the split's, each read once and straight into
//                 registers (16 loads of 16 bytes per lane, the next block's issued as soon as the present one's are
//                 used), and runs on v_mfma_f32_16x16x32_f16
//                   scores^T  (16 tokens x 16 columns)  A = codes of 16 tokens as fp16 numbers, B = the query rows,
//                   softmax per lane (its column, 16 of the block's 64 tokens), running offset in the log2 domain,
//                   out^T    (16 dims x 16 columns) += A = codes of 16 dims, B = the weights from the lane's registers.
//                 A code becomes an fp16 number exactly (one v_perm and one packed subtraction for two), so the products
//                 are those of whole numbers with fp16 queries / weights, summed in fp32.
//                 The key scale multiplies the score.  The value scale enters the weight's exponent: with
//                   p'_t = 2^(s_t + log2(vscale) - m),  out = sum p'_t code_t / sum p'_t / vscale,
//                 so neither the codes nor the sums need a multiplication, and m follows the largest s + log2(vscale).
//                 Weights are rounded to fp16 (2^-12 of each) for the product; their sum is of the unrounded ones.
//   combine       joins the splits' (offset, sum, rows) in fp32.
// Bound by memory: 16 KB a block and head.
//
// Selection (lkv_kv8_select_blocks): a score per finished block, the upper bound sum_d max(q8 lo, q8 hi) of the product
// with any of its keys, from the per-dim lowest and highest codes (256 bytes a block) and the query rows in 8 bits, on
// v_mfma_i32_16x16x64_i8: max(q8 lo, q8 hi) = min(q8, 0) lo + max(q8, 0) hi.  The sum is a whole number below 2^24, so a
// score has two roundings (the query's scale, the block's) whatever the order of the work, and the choice is the same
// everywhere.  Then a radix selection per (sequence, kv head).
#include "kv8_common.h"

namespace lkv {
namespace kv8 {

int check_store(const lkv_kv8_store* s, const char* what);
Store device_store(const lkv_kv8_store* s);
int check_rows(const void* x, const int64_t* strides, int dtype, const char* what, const char* name);

namespace {

constexpr int kThr = 256;
constexpr int kWaves = 4;
constexpr int kManyCols = 256;  // columns of a workgroup of the many-row kernel
constexpr int kManyChunk = 8;   // and the fewest blocks that a split of it gets

__device__ __forceinline__ f32x4 mfma16(const f16x8& a, const f16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ int lane_i(int v, int l) { return __builtin_amdgcn_readlane(v, l); }

struct SplitArgs {
  Store st;
  Rows r;
  const int* index;  // [B][Hkv][n_index] chosen blocks (-1: none), or null: all
  int n_index;
  int groups, chunk, splits;
  float* part_o;   // [B][Hkv][cols][splits][128]
  float* part_ml;  // [B][Hkv][cols][splits][2]
};

// Writes row `col` of (b, h), dims d .. d + 3.
template <int DT>
__device__ __forceinline__ void store_row(const Rows& r, int b, int h, int col, int d, const f32x4& o) {
  const int s = col / r.G, g = col - s * r.G;
  store4<DT>(r.out, b * r.o_sb + static_cast<int64_t>(h * r.G + g) * r.o_sh + s * r.o_ss + d, o[0], o[1], o[2], o[3]);
}

template <int DT, int NT>
__global__ __launch_bounds__(kThr, 2) void split_kernel(SplitArgs P) {
  constexpr int kRow = kD + 4;  // floats of a staged row
  __shared__ __align__(16) float s_o[kWaves][16][kRow];
  __shared__ float s_m[kWaves][16 * NT], s_l[kWaves][16 * NT];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const Store& st = P.st;
  const Rows& r = P.r;
  const int b = blockIdx.z, h = blockIdx.y / P.groups, group = blockIdx.y - h * P.groups;
  const int len = min(max(r.lens[b], 0), r.max_len);
  const int qlen = min(r.q_lens ? min(max(r.q_lens[b], 0), r.S) : r.S, len);
  const int nfull = len / kBlk, rest = len - nfull * kBlk;
  const int64_t bh = static_cast<int64_t>(b) * st.Hkv + h;
  // units: the blocks (or list entries), then the unfinished block
  const int nlist = P.index ? P.n_index : nfull;
  const int units = nlist + (rest ? 1 : 0);
  const int u0 = blockIdx.x * P.chunk;
  const int col0 = group * 16 * NT;
  if (P.splits > 1 && u0 >= units) {  // nothing to do: an empty record
    const int col = col0 + tid;
    if (tid < 16 * NT && col < r.cols)
      *reinterpret_cast<float2*>(P.part_ml + 2 * ((bh * r.cols + col) * P.splits + blockIdx.x)) = float2{-INFINITY, 0.f};
    return;
  }
  const int u1 = min(u0 + P.chunk, units);

  // ---- query rows: lane: column c16, dims 64 (ks / 2) + 16 g + 8 (ks % 2) + j
  f16x8 qf[NT][4];
  int lim[NT];  // tokens that the lane's column sees (all, if there is no such row)
  float m[NT], l[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = col0 + 16 * n + c16, s = col / r.G, hq = col - s * r.G;
    const bool ok = col < r.cols && s < qlen;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      qf[n][ks] = f16x8{};
      if (ok)
        qf[n][ks] = load_q8<DT>(r.q, b * r.q_sb + static_cast<int64_t>(h * r.G + hq) * r.q_sh + s * r.q_ss +
                                         64 * (ks >> 1) + 16 * g + 8 * (ks & 1));
    }
    lim[n] = ok ? len - qlen + s + 1 : 0x7fffffff;
    m[n] = ok ? -INFINITY : 0.f;  // a column that is no row keeps offset 0 over zero scores
    l[n] = 0.f;
  }
  const int lim_min = len - qlen + col0 / r.G + 1;  // columns' queries ascend
  f32x4 o[NT][8];  // column c16, dims 16 jt + 4 g + i
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int jt = 0; jt < 8; ++jt) o[n][jt] = f32x4{0.f, 0.f, 0.f, 0.f};

  // One block: kf(T, ks), vf(jt, ks) give the operands, kc = key scale * scale * log2(e), lv = log2(value scale),
  // iv = 1 / value scale; tokens from `left` on (relative to a column's limit) are hidden.
  // next() issues the next block's key loads once this block's keys are used.
  auto step = [&](auto kf, auto vf, float kc, float lv, float iv, int t0, auto next) {
    f32x4 sc[NT][4];
#pragma unroll
    for (int T = 0; T < 4; ++T) {
      f16x8 a[4];
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) a[ks] = kf(T, ks);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        sc[n][T] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) sc[n][T] = mfma16(a[ks], qf[n][ks], sc[n][T]);
      }
    }
    next();
    f16x8 pf[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float s[16];
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = fmaf(sc[n][e >> 2][e & 3], kc, lv - m[n]);
        mx = fmaxf(mx, s[e]);
      }
      if (t0 + kBlk > lim_min || wave_ballot(mx > kMaxWeight) != 0) {  // uniform
        const int left = lim[n] - t0 - 4 * g;  // the lane's token 16 T + i is visible below this
        mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = fmaf(sc[n][e >> 2][e & 3], kc, lv);
          s[e] = 16 * (e >> 2) + (e & 3) < left ? x : -INFINITY;
          mx = fmaxf(mx, s[e]);
        }
        mx = groups_max(mx);
        const float mn = mx - m[n] > kMaxWeight ? mx - kTopWeight : m[n];
        const float mu = mn == -INFINITY ? 0.f : mn;
        const float alpha = exp2_(m[n] - mu);
        m[n] = mn;
        l[n] *= alpha;
#pragma unroll
        for (int jt = 0; jt < 8; ++jt) o[n][jt] *= alpha;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] -= mu;
      }
      float ps = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = exp2_(s[e]);
        ps += s[e];
      }
      l[n] = fmaf(ps, iv, l[n]);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        pf[n][ks] = __builtin_bit_cast(f16x8, u32x4{pk2(s[8 * ks], s[8 * ks + 1]), pk2(s[8 * ks + 2], s[8 * ks + 3]),
                                                    pk2(s[8 * ks + 4], s[8 * ks + 5]), pk2(s[8 * ks + 6], s[8 * ks + 7])});
    }
#pragma unroll
    for (int jt = 0; jt < 8; ++jt)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const f16x8 a = vf(jt, ks);
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][jt] = mfma16(a, pf[n][ks], o[n][jt]);
      }
  };

  // ---- the wave's units u0 + wave, + kWaves, ...: lane i holds number i's block and scales, 64 at a time
  const int* list = P.index ? P.index + bh * P.n_index : nullptr;
  const uint8_t* kbase = st.k_codes + bh * st.blocks * kBlkBytes + c16 * kD + 16 * g;
  const uint8_t* vbase = st.v_codes + bh * st.blocks * kBlkBytes + c16 * kBlk + 16 * g;
  u32x4 kr[8], vr[8];
  auto load_k = [&](int blk) {
    const uint8_t* p = kbase + static_cast<int64_t>(blk) * kBlkBytes;
#pragma unroll
    for (int j = 0; j < 8; ++j) kr[j] = *reinterpret_cast<const u32x4*>(p + (j >> 1) * 16 * kD + (j & 1) * 64);
  };
  auto load_v = [&](int blk) {
    const uint8_t* p = vbase + static_cast<int64_t>(blk) * kBlkBytes;
#pragma unroll
    for (int j = 0; j < 8; ++j) vr[j] = *reinterpret_cast<const u32x4*>(p + j * 16 * kBlk);
  };
  const int uend = min(u1, nlist);
  for (int ub = u0 + wave; ub < uend; ub += 64 * kWaves) {
    const int mine = ub + kWaves * lane;
    int blk_l = -1;
    if (mine < uend) {
      blk_l = list ? list[mine] : mine;
      if (blk_l >= nfull) blk_l = -1;  // (no such block: skipped)
    }
    float ks_l = 0.f, vs_l = kMinScale;
    if (blk_l >= 0) {
      const float2 sc = *reinterpret_cast<const float2*>(st.scales + 2 * (bh * st.blocks + blk_l));
      ks_l = sc.x;
      vs_l = fmaxf(sc.y, kMinScale);
    }
    const float kc_l = ks_l * r.scale_log2, lv_l = __log2f(vs_l), iv_l = 1.f / vs_l;
    // skipped entries lie anywhere in a list: only those lanes that hold a block are walked
    uint64_t todo = wave_ballot(blk_l >= 0);
    if (!todo) continue;
    int i = __builtin_ctzll(todo);
    int blk = lane_i(blk_l, i);
    load_k(blk);
    load_v(blk);
    while (true) {
      todo &= todo - 1;
      const float kc = lane_f(kc_l, i), lv = lane_f(lv_l, i), iv = lane_f(iv_l, i);
      const int t0 = blk * kBlk;
      const bool more = todo != 0;
      if (more) i = __builtin_ctzll(todo), blk = lane_i(blk_l, i);
      step([&](int T, int ks) { return codes8h(kr[2 * T + (ks >> 1)][2 * (ks & 1)], kr[2 * T + (ks >> 1)][2 * (ks & 1) + 1]); },
           [&](int jt, int ks) { return codes8h(vr[jt][2 * ks], vr[jt][2 * ks + 1]); }, kc, lv, iv, t0,
           [&]() { if (more) load_k(blk); });
      if (!more) break;
      load_v(blk);
    }
  }
  // ---- the unfinished block, by the wave whose turn it is
  if (rest && u1 == units && (nlist - u0) % kWaves == wave) {
    const uint16_t* kt = st.k_tail + bh * kBlkBytes + c16 * kD + 16 * g;
    const uint16_t* vt = st.v_tail + bh * kBlkBytes + c16 * kBlk + 16 * g;
    step(
        [&](int T, int ks) {
          return *reinterpret_cast<const f16x8*>(kt + T * 16 * kD + 64 * (ks >> 1) + 8 * (ks & 1));
        },
        [&](int jt, int ks) {
          // (slots past the last token keep older values, finite ones: their weight is 0)
          return *reinterpret_cast<const f16x8*>(vt + jt * 16 * kBlk + 8 * ks);
        },
        r.scale_log2, 0.f, 1.f, nfull * kBlk, [] {});
  }

  // ---- join the waves, one 16-column tile at a time
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    l[n] = groups_sum(l[n]);
    if (g == 0) {
      s_m[wave][16 * n + c16] = m[n];
      s_l[wave][16 * n + c16] = l[n];
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (n) __syncthreads();
#pragma unroll
    for (int jt = 0; jt < 8; ++jt) *reinterpret_cast<f32x4*>(&s_o[wave][c16][16 * jt + 4 * g]) = o[n][jt];
    __syncthreads();
    const int row = tid >> 4, d = 4 * (tid & 15);
    const int col = col0 + 16 * n + row;
    if (col < r.cols) {
      float M = s_m[0][16 * n + row];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) M = fmaxf(M, s_m[w][16 * n + row]);
      const float mu = M == -INFINITY ? 0.f : M;
      f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
      float L = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float a = exp2_(s_m[w][16 * n + row] - mu);
        L += a * s_l[w][16 * n + row];
        acc[0] += a * *reinterpret_cast<const f32x4*>(&s_o[w][row][d]);
        acc[1] += a * *reinterpret_cast<const f32x4*>(&s_o[w][row][64 + d]);
      }
      const bool row_ok = col / r.G < qlen;
      if (P.splits == 1) {
        const bool some = row_ok && L != 0.f;  // no such row, or no token: zeros
        const float inv = some ? 1.f / L : 0.f;
        if (!some) acc[0] = acc[1] = f32x4{0.f, 0.f, 0.f, 0.f};
        store_row<DT>(r, b, h, col, d, acc[0] * inv);
        store_row<DT>(r, b, h, col, 64 + d, acc[1] * inv);
      } else {
        const int64_t at = ((bh * r.cols + col) * P.splits + blockIdx.x);
        *reinterpret_cast<f32x4*>(P.part_o + at * kD + d) = acc[0];
        *reinterpret_cast<f32x4*>(P.part_o + at * kD + 64 + d) = acc[1];
        if ((tid & 15) == 0)
          *reinterpret_cast<float2*>(P.part_ml + 2 * at) = row_ok ? float2{M, L} : float2{-INFINITY, 0.f};
      }
    }
  }
}

struct CombineArgs {
  Rows r;
  const float* part_o;
  const float* part_ml;
  int Hkv, splits;
};

// One workgroup per row: 8 groups of 32 lanes, each every 8th split, 4 dims a lane.  A split without a token for the row
// has offset -inf (and wrote no sums).
template <int DT>
__global__ __launch_bounds__(kThr) void combine_kernel(CombineArgs P) {
  __shared__ __align__(16) float s_o[8][kD];
  __shared__ float s_l[8];
  const Rows& r = P.r;
  const int tid = threadIdx.x, d = 4 * (tid & 31), part = tid >> 5;
  const int64_t row = blockIdx.x;  // ((sequence, kv head), column)
  const int n = P.splits;
  const float* ml = P.part_ml + row * n * 2;
  const float* po = P.part_o + row * n * kD + d;
  float M = -INFINITY;
  for (int i = tid & 63; i < n; i += 64) M = fmaxf(M, ml[2 * i]);  // every wave for itself
  M = wave_max(M);
  const float mu = M == -INFINITY ? 0.f : M;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  float L = 0.f;
#pragma unroll 4
  for (int i = part; i < n; i += 8) {
    const float2 x = *reinterpret_cast<const float2*>(ml + 2 * i);
    const f32x4 v = *reinterpret_cast<const f32x4*>(po + static_cast<int64_t>(i) * kD);
    if (x.x != -INFINITY) {
      const float a = exp2_(x.x - mu);
      L += a * x.y;
      acc += a * v;
    }
  }
  *reinterpret_cast<f32x4*>(&s_o[part][d]) = acc;
  if ((tid & 31) == 0) s_l[part] = L;
  __syncthreads();
  if (part == 0) {
#pragma unroll
    for (int p = 1; p < 8; ++p) {
      acc += *reinterpret_cast<const f32x4*>(&s_o[p][d]);
      L += s_l[p];
    }
    const float inv = L != 0.f ? 1.f / L : 0.f;
    if (L == 0.f) acc = f32x4{0.f, 0.f, 0.f, 0.f};
    const int64_t bh = row / r.cols;
    store_row<DT>(r, static_cast<int>(bh / P.Hkv), static_cast<int>(bh % P.Hkv), static_cast<int>(row - bh * r.cols), d,
                  acc * inv);
  }
}

// --------------------------------------------------------------------------------------------------- block selection
constexpr int kSelThr = 256;
constexpr int kLdsKeys = 8192;  // so many keys of a (sequence, kv head) stay in LDS, more are read again from memory

struct SelectArgs {
  Store st;
  const void* q;
  int64_t q_sb, q_sh;
  const int* lens;
  int G, n, sink, recent;
  int max_blocks;   // the grid's bound on finished blocks
  uint32_t* keys;   // [B][Hkv][max_blocks]
  int* index;       // [B][Hkv][n]
};

// Order-preserving bits of a score (-0 made +0 before); larger is larger.
__device__ __forceinline__ uint32_t sort_bits(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Scores of 16 blocks per wave and step; a lane has column c16 = query head, k slots 16 g + j of a 64-dim step.
template <int DT>
__global__ __launch_bounds__(kThr) void score_kernel(SelectArgs P) {
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const int h = blockIdx.y, b = blockIdx.z;
  const Store& st = P.st;
  const int len = min(max(P.lens[b], 0), st.blocks * kBlk);
  const int nfull = min(len / kBlk, P.max_blocks);
  const int64_t bh = static_cast<int64_t>(b) * st.Hkv + h;
  const int step = gridDim.x * kWaves * 16;
  for (int j0 = (blockIdx.x * kWaves + wave) * 16; j0 < nfull; j0 += step) {
    const int jr = min(j0 + c16, nfull - 1);
    i32x4 a[4];
    const int8_t* p = st.ranges + (bh * st.blocks + jr) * 2 * kD + 16 * g;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) a[ks] = *reinterpret_cast<const i32x4*>(p + 64 * ks);
    float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    for (int h0 = 0; h0 < P.G; h0 += 16) {
      // the column's query in 8 bits: dims 16 g .. + 15 and 64 + 16 g .. + 15
      const bool ok = h0 + c16 < P.G;
      float x[4][8];
      float amax = 0.f;
      const int64_t at = b * P.q_sb + static_cast<int64_t>(h * P.G + (ok ? h0 + c16 : 0)) * P.q_sh + 16 * g;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        load8<DT>(P.q, at + 64 * (k >> 1) + 8 * (k & 1), x[k]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[k][j] = h2f(f2h(clamp_kv(x[k][j])));
          amax = fmaxf(amax, fabsf(x[k][j]));
        }
      }
      amax = groups_max(amax);
      const float inv = code_factor(amax), qs = amax * kStep;
      i32x4 neg[2], pos[2];
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        uint32_t un = 0, up = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int q8 = static_cast<int>(rintf(x[w >> 1][4 * (w & 1) + j] * inv));
          un |= (static_cast<uint32_t>(min(q8, 0)) & 0xffu) << (8 * j);
          up |= (static_cast<uint32_t>(max(q8, 0)) & 0xffu) << (8 * j);
        }
        neg[w >> 2][w & 3] = static_cast<int>(un);
        pos[w >> 2][w & 3] = static_cast<int>(up);
      }
      i32x4 d = i32x4{0, 0, 0, 0};
      d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[0], neg[0], d, 0, 0, 0);
      d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[1], neg[1], d, 0, 0, 0);
      d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[2], pos[0], d, 0, 0, 0);
      d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[3], pos[1], d, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) best[i] = fmaxf(best[i], row16_max(ok ? static_cast<float>(d[i]) * qs : -INFINITY));
    }
    // rows (blocks) j0 + 4 g + i; lane c16 = i writes it
    const float mine = c16 == 0 ? best[0] : c16 == 1 ? best[1] : c16 == 2 ? best[2] : best[3];
    const int j = j0 + 4 * g + c16;
    if (c16 < 4 && j < nfull) {
      uint32_t key = sort_bits(mine * st.scales[2 * (bh * st.blocks + j)]);
      if (j < P.sink || j >= nfull - P.recent) key = 0xffffffffu;
      P.keys[bh * P.max_blocks + j] = key;
    }
  }
}

// The n highest keys of a (sequence, kv head), equal ones by index, as ascending indices; the rest of the row is -1.
__global__ __launch_bounds__(kSelThr) void select_kernel(SelectArgs P) {
  __shared__ uint32_t s_key[kLdsKeys];
  __shared__ uint32_t s_hist[256];
  __shared__ uint32_t s_pick[2];
  __shared__ int s_cnt[2][kSelThr / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x, b = blockIdx.y;
  const Store& st = P.st;
  const int len = min(max(P.lens[b], 0), st.blocks * kBlk);
  const int nfull = min(len / kBlk, P.max_blocks);
  const int64_t bh = static_cast<int64_t>(b) * st.Hkv + h;
  int* out = P.index + bh * P.n;
  if (nfull <= P.n) {  // all of them
    for (int j = tid; j < P.n; j += kSelThr) out[j] = j < nfull ? j : -1;
    return;
  }
  const uint32_t* keys = P.keys + bh * P.max_blocks;
  const bool in_lds = nfull <= kLdsKeys;
  if (in_lds)
    for (int j = tid; j < nfull; j += kSelThr) s_key[j] = keys[j];  // (a thread reads back its own)
  auto key_at = [&](int j) { return in_lds ? s_key[j] : keys[j]; };
  // radix selection from the top byte down: the key of rank n is (prefix, low bits)
  uint32_t prefix = 0;
  int need = P.n;  // rank within the keys that share the prefix
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    s_hist[tid] = 0;
    __syncthreads();
    const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    for (int j = tid; j < nfull; j += kSelThr) {
      const uint32_t k = key_at(j);
      if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (wave == 0) {
      // lane: bins 4 lane .. + 3; counts above them
      uint32_t c[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = s_hist[4 * lane + i], sum += c[i];
      uint32_t above = sum;  // inclusive sum from lane on, then exclusive
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const uint32_t t = __shfl_down(above, off);
        if (lane + off < 64) above += t;
      }
      above -= sum;
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        if (above < static_cast<uint32_t>(need) && above + c[i] >= static_cast<uint32_t>(need)) {
          s_pick[0] = 4 * lane + i;
          s_pick[1] = above;
        }
        above += c[i];
      }
    }
    __syncthreads();
    prefix |= s_pick[0] << shift;
    need -= static_cast<int>(s_pick[1]);
  }
  // keys above `prefix` and the first `need` equal to it, in index order
  int base_gt = 0, base_eq = 0;
  for (int j0 = 0; j0 < nfull; j0 += kSelThr) {
    const int j = j0 + tid;
    const uint32_t k = j < nfull ? key_at(j) : 0u;
    const bool gt = j < nfull && k > prefix, eq = j < nfull && k == prefix;
    const uint64_t mg = wave_ballot(gt), me = wave_ballot(eq);
    if (lane == 0) {
      s_cnt[0][wave] = __popcll(mg);
      s_cnt[1][wave] = __popcll(me);
    }
    __syncthreads();
    int gt_before = base_gt + lane_prefix(mg), eq_before = base_eq + lane_prefix(me);
#pragma unroll
    for (int w = 0; w < kSelThr / 64; ++w) {
      if (w < wave) {
        gt_before += s_cnt[0][w];
        eq_before += s_cnt[1][w];
      }
      base_gt += s_cnt[0][w];
      base_eq += s_cnt[1][w];
    }
    if (gt || (eq && eq_before < need)) out[gt_before + min(eq_before, need)] = j;
    __syncthreads();
  }
}

}  // namespace

Plan make_plan(int64_t B, int64_t Hkv, int64_t cols, int64_t units) {
  Plan p;
  if (units < 1) units = 1;
  const int64_t cus = device_cu_count();
  p.nt = cols <= 16 ? 1 : cols <= 64 ? 2 : 0;
  const int64_t wide = p.nt ? 16 * p.nt : kManyCols;
  p.groups = static_cast<int>((cols + wide - 1) / wide);
  const int64_t items = B * Hkv * p.groups;
  // workgroups resident at once: two of the few-row kernel on a CU, one of the other
  int64_t want = ((p.nt ? 2 : 1) * cus + items - 1) / items;
  int64_t chunk = (units + want - 1) / want;
  const int64_t unit = p.nt ? kWaves : 2;  // a block for every wave, or a pair of blocks
  chunk = (chunk + unit - 1) / unit * unit;
  if (!p.nt && chunk < kManyChunk) chunk = kManyChunk;
  p.chunk = static_cast<int>(chunk);
  p.splits = static_cast<int>((units + chunk - 1) / chunk);
  return p;
}

size_t plan_bytes(const Plan& p, int64_t B, int64_t Hkv, int64_t cols) {
  return p.splits > 1 ? static_cast<size_t>(B * Hkv * cols) * p.splits * (kD + 2) * sizeof(float) : 0;
}

namespace {

template <int DT>
void launch_split(const SplitArgs& P, int nt, int64_t B, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(P.splits), static_cast<unsigned>(P.st.Hkv * P.groups), static_cast<unsigned>(B));
  if (nt == 1)
    hipLaunchKernelGGL((split_kernel<DT, 1>), grid, dim3(kThr), 0, st, P);
  else
    hipLaunchKernelGGL((split_kernel<DT, 2>), grid, dim3(kThr), 0, st, P);
}

int64_t units_of(int64_t max_len, int64_t n_index) {
  return n_index > 0 ? n_index + 1 : (max_len + kBlk - 1) / kBlk;
}

int check_attn(const lkv_kv8_store* store, int64_t Hq, int64_t S, int64_t max_len, const char* what) {
  if (int rc = check_store(store, what)) return rc;
  LKV_REQUIRE(Hq > 0 && Hq % store->kv_heads == 0, "%s: %lld query heads over %lld kv heads", what, (long long)Hq,
              (long long)store->kv_heads);
  LKV_REQUIRE(S >= 0 && S < (1ll << 24) && Hq / store->kv_heads * S < (1ll << 30), "%s: S=%lld out of range", what,
              (long long)S);
  LKV_REQUIRE(max_len >= 0 && max_len <= store->blocks * kBlk, "%s: max_len=%lld outside a store of %lld tokens", what,
              (long long)max_len, (long long)(store->blocks * kBlk));
  return LKV_OK;
}

}  // namespace
}  // namespace kv8
}  // namespace lkv

using namespace lkv;
using namespace lkv::kv8;

extern "C" size_t lkv_kv8_attn_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t S, int64_t max_len,
                                               int64_t n_index) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || S <= 0 || max_len < 0 || n_index < 0) return 0;
  const int64_t cols = Hq / Hkv * S;
  return plan_bytes(make_plan(B, Hkv, cols, units_of(max_len, n_index)), B, Hkv, cols);
}

extern "C" int lkv_kv8_attn(const lkv_kv8_store* store, const void* q, const int64_t* q_strides, int dtype, int64_t Hq,
                            int64_t S, const int32_t* lens, const int32_t* q_lens, int64_t max_len,
                            const int32_t* index, int64_t n_index, float scale, void* out, const int64_t* out_strides,
                            void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_attn(store, Hq, S, max_len, "kv8_attn")) return rc;
  LKV_REQUIRE(dtype == LKV_DTYPE_F32 || dtype == LKV_DTYPE_F16 || dtype == LKV_DTYPE_BF16, "kv8_attn: dtype %d", dtype);
  LKV_REQUIRE(n_index >= 0 && n_index < (1ll << 24) && (n_index == 0) == (index == nullptr),
              "kv8_attn: a list of %lld blocks", (long long)n_index);
  LKV_REQUIRE(!index || S == 1, "kv8_attn: a block list is for one query per sequence");
  const int64_t B = store->batch, Hkv = store->kv_heads, G = Hq / Hkv, cols = G * S;
  LKV_REQUIRE(B * Hkv * cols < (1ll << 31), "kv8_attn: %lld query rows", (long long)(B * Hkv * cols));
  if (B == 0 || S == 0) return LKV_OK;
  LKV_REQUIRE(q && out && lens, "kv8_attn: null pointer");
  if (int rc = check_rows(q, q_strides, dtype, "kv8_attn", "q")) return rc;
  if (int rc = check_rows(out, out_strides, dtype, "kv8_attn", "out")) return rc;
  Plan p = make_plan(B, Hkv, cols, units_of(max_len, n_index));
  const size_t need = plan_bytes(p, B, Hkv, cols);
  LKV_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
              "kv8_attn: workspace of %zu bytes (16-byte aligned) required, got %zu", need, workspace_bytes);
  Rows r;
  r.q = q;
  r.q_sb = q_strides[0];
  r.q_sh = q_strides[1];
  r.q_ss = q_strides[2];
  r.out = out;
  r.o_sb = out_strides[0];
  r.o_sh = out_strides[1];
  r.o_ss = out_strides[2];
  r.lens = lens;
  r.q_lens = q_lens;
  r.G = static_cast<int>(G);
  r.S = static_cast<int>(S);
  r.cols = static_cast<int>(cols);
  r.max_len = static_cast<int>(max_len);
  r.scale_log2 = scale * kLog2e;
  hipStream_t st = static_cast<hipStream_t>(stream);
  float* part_o = static_cast<float*>(workspace);
  float* part_ml = part_o + static_cast<size_t>(B * Hkv * cols) * p.splits * kD;
  SplitArgs A{device_store(store), r, index, static_cast<int>(n_index), p.groups, p.chunk, p.splits, part_o, part_ml};
  if (!p.nt) {
    if (int rc = launch_prefill(A.st, r, p, dtype, B, part_o, part_ml, st)) return rc;
  } else {
    if (dtype == LKV_DTYPE_F32)
      launch_split<LKV_DTYPE_F32>(A, p.nt, B, st);
    else if (dtype == LKV_DTYPE_F16)
      launch_split<LKV_DTYPE_F16>(A, p.nt, B, st);
    else
      launch_split<LKV_DTYPE_BF16>(A, p.nt, B, st);
    LKV_LAUNCH_CHECK("kv8_attn split");
  }
  if (p.splits > 1) {
    const CombineArgs C{r, part_o, part_ml, static_cast<int>(Hkv), p.splits};
    const dim3 grid(static_cast<unsigned>(B * Hkv * cols));
    if (dtype == LKV_DTYPE_F32)
      hipLaunchKernelGGL(combine_kernel<LKV_DTYPE_F32>, grid, dim3(kThr), 0, st, C);
    else if (dtype == LKV_DTYPE_F16)
      hipLaunchKernelGGL(combine_kernel<LKV_DTYPE_F16>, grid, dim3(kThr), 0, st, C);
    else
      hipLaunchKernelGGL(combine_kernel<LKV_DTYPE_BF16>, grid, dim3(kThr), 0, st, C);
    LKV_LAUNCH_CHECK("kv8_attn combine");
  }
  return LKV_OK;
}

extern "C" size_t lkv_kv8_select_workspace_bytes(int64_t B, int64_t Hkv, int64_t max_len) {
  if (B <= 0 || Hkv <= 0 || max_len < 0) return 0;
  return static_cast<size_t>(B * Hkv * (max_len / kBlk)) * sizeof(uint32_t);
}

extern "C" int lkv_kv8_select_blocks(const lkv_kv8_store* store, const void* q, const int64_t* q_strides, int dtype,
                                     int64_t Hq, const int32_t* lens, int64_t max_len, int64_t n, int64_t sink,
                                     int64_t recent, int32_t* index, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  if (int rc = check_attn(store, Hq, 1, max_len, "kv8_select_blocks")) return rc;
  LKV_REQUIRE(dtype == LKV_DTYPE_F32 || dtype == LKV_DTYPE_F16 || dtype == LKV_DTYPE_BF16,
              "kv8_select_blocks: dtype %d", dtype);
  LKV_REQUIRE(n >= 1 && n < (1ll << 24) && sink >= 0 && recent >= 0 && sink + recent <= n,
              "kv8_select_blocks: %lld blocks with the first %lld and the last %lld among them", (long long)n,
              (long long)sink, (long long)recent);
  const int64_t mb = max_len / kBlk;
  const int64_t B = store->batch, Hkv = store->kv_heads;
  if (B == 0) return LKV_OK;
  LKV_REQUIRE(q && lens && index, "kv8_select_blocks: null pointer");
  if (int rc = check_rows(q, q_strides, dtype, "kv8_select_blocks", "q")) return rc;
  const size_t need = lkv_kv8_select_workspace_bytes(B, Hkv, max_len);
  LKV_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned4(workspace))),
              "kv8_select_blocks: workspace of %zu bytes required, got %zu", need, workspace_bytes);
  SelectArgs P;
  P.st = device_store(store);
  P.q = q;
  P.q_sb = q_strides[0];
  P.q_sh = q_strides[1];
  P.lens = lens;
  P.G = static_cast<int>(Hq / Hkv);
  P.n = static_cast<int>(n);
  P.sink = static_cast<int>(sink);
  P.recent = static_cast<int>(recent);
  P.max_blocks = static_cast<int>(mb);
  P.keys = static_cast<uint32_t*>(workspace);
  P.index = index;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (mb > n) {  // otherwise every block is chosen
    const int64_t tiles = (mb + 16 * kWaves - 1) / (16 * kWaves);
    const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(Hkv), static_cast<unsigned>(B));
    if (dtype == LKV_DTYPE_F32)
      hipLaunchKernelGGL(score_kernel<LKV_DTYPE_F32>, grid, dim3(kThr), 0, st, P);
    else if (dtype == LKV_DTYPE_F16)
      hipLaunchKernelGGL(score_kernel<LKV_DTYPE_F16>, grid, dim3(kThr), 0, st, P);
    else
      hipLaunchKernelGGL(score_kernel<LKV_DTYPE_BF16>, grid, dim3(kThr), 0, st, P);
    LKV_LAUNCH_CHECK("kv8_select_blocks score");
  }
  hipLaunchKernelGGL(select_kernel, dim3(static_cast<unsigned>(Hkv), static_cast<unsigned>(B)), dim3(kSelThr), 0,
                     st, P);
  LKV_LAUNCH_CHECK("kv8_select_blocks");
  return LKV_OK;
}
