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
// Bound by memory where there are many blocks: 16 KB a block and head, one 4-wave workgroup a CU with all of a block's 16
// loads of a wave in flight.  1 x 131072 tokens (32/8 heads, 269 MB): 45 us the split kernel (6.0 TB/s; a plain read loop
// 6.0-6.3), 51-53 us a call; 32 x 8192: 90-92 us (5.9 TB/s); 32 sequences of 1.6-8 K tokens 68 us, the longest of them bounds
// it.  8 waves were no faster, nontemporal loads gained 5 % there and lost as much with many sequences.
// The work is split for max_len, not for the lengths: 1 x 4133 tokens take 12 us a call with max_len (or a store) of up to
// 8192, 13 with 32768 and 31 with 131072, where two splits hold all of them.  From one (sequence, kv head) pair a CU on a pair
// is one workgroup's: 32 sequences of which one has 131072 tokens and the others 2048 take 770 us.
// Bound by latency where there are few: 1 x 4133 tokens 9.2-9.8 us in a replayed graph, 5.5 the split kernel (length, then
// loads, then one block's 440 vector instructions, then the join) and 3.5 the combine.  5 queries of 8 x 4096 tokens: four
// blocks a wave, 16.3 us traced, of which vector work is 38 % and products 13 %; what starts and ends a split is not covered.
//
// Selection (lkv_kv8_select_blocks): a score per finished block, the upper bound sum_d max(q8 lo, q8 hi) of the product
// with any of its keys, from the per-dim lowest and highest codes (256 bytes a block) and the query rows in 8 bits, on
// v_mfma_i32_16x16x64_i8: max(q8 lo, q8 hi) = min(q8, 0) lo + max(q8, 0) hi.  The sum is a whole number below 2^24, so a
// score has two roundings (the query's scale, the block's) whatever the order of the work, and the choice is the same
// everywhere.  Then a selection per (sequence, kv head), by the same workgroup up to 512 blocks: by counting up to 128, by
// radix passes beyond.  Bound by latency: 128 blocks 6.0 us a call in a replayed graph, 300 of 16 sequences 8.7 us; 2048
// blocks 10.2 us, the scores in a launch of their own.
#include "kv8_common.h"

namespace lkv {
namespace kv8 {

int check_store(const lkv_kv8_store* s, const char* what);
Store device_store(const lkv_kv8_store* s);
int check_rows(const void* x, const int64_t* strides, int dtype, const char* what, const char* name);

namespace {

constexpr int kThr = 256;
constexpr int kWaves = 4;  // of a split workgroup
constexpr int kOneSplit = 3 * kWaves;  // so few units are one split
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
  // the columns' query rows, asked for first (a column that is no row reads the last one)
  const int col0 = group * 16 * NT;
  RawQ<DT> qraw[NT][4];
  int qs[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = min(col0 + 16 * n + c16, r.cols - 1);
    qs[n] = col / r.G;
    const int64_t at = b * r.q_sb + static_cast<int64_t>(h * r.G + col - qs[n] * r.G) * r.q_sh + qs[n] * r.q_ss + 16 * g;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) qraw[n][ks] = load_raw_q8<DT>(r.q, at + 64 * (ks >> 1) + 8 * (ks & 1));
  }
  const int len = held_tokens(r.lens[b], r.max_len);
  const int qlen = min(r.q_lens ? min(max(r.q_lens[b], 0), r.S) : r.S, len);
  const int nfull = len / kBlk, rest = len - nfull * kBlk;
  const int64_t bh = static_cast<int64_t>(b) * st.Hkv + h;
  // units: the blocks (or list entries), then the unfinished block
  const int nlist = P.index ? P.n_index : nfull;
  const int units = nlist + (rest ? 1 : 0);
  const int u0 = blockIdx.x * P.chunk;
  if (P.splits > 1 && u0 >= units) {  // nothing to do: an empty record
    const int col = col0 + tid;
    if (tid < 16 * NT && col < r.cols)
      *reinterpret_cast<float2*>(P.part_ml + 2 * ((bh * r.cols + col) * P.splits + blockIdx.x)) = part_record(-INFINITY, 0.f);
    return;
  }
  const int u1 = min(u0 + P.chunk, units);

  // ---- the wave's units u0 + wave, + kWaves, ...: lane i holds number i's block and factors, 64 at a time
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
  const int uend = min(u0 + P.chunk, nlist);
  int ub = u0 + wave, i = 0, blk = 0;
  uint64_t todo = 0;  // lanes whose blocks are still to do (skipped entries lie anywhere in a list)
  int blk_l;
  float2 scale_l;
  // the next 64 units that hold a block; its first one's loads are on their way afterwards
  auto next_units = [&]() {
    for (; ub < uend && !todo; ub += 64 * kWaves) {
      const int mine = ub + kWaves * lane;
      blk_l = -1;
      if (mine < uend) {
        blk_l = list ? list[mine] : mine;
        if (blk_l >= nfull) blk_l = -1;  // (no such block)
      }
      scale_l = float2{0.f, 0.f};
      if (blk_l >= 0) scale_l = *reinterpret_cast<const float2*>(st.scales + 2 * (bh * st.blocks + blk_l));
      todo = wave_ballot(blk_l >= 0);
    }
    if (todo) {
      i = __builtin_ctzll(todo);
      blk = lane_i(blk_l, i);
      load_k(blk);
      load_v(blk);
    }
  };
  next_units();

  // ---- the queries' rows: lane: column c16, dims 64 (ks / 2) + 16 g + 8 (ks % 2) + j
  f16x8 qf[NT][4];
  int lim[NT];  // tokens that the lane's column sees (all, if there is no such row)
  float m[NT], l[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const bool ok = col0 + 16 * n + c16 < r.cols && qs[n] < qlen;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) qf[n][ks] = ok ? convert_q8<DT>(qraw[n][ks]) : f16x8{};
    lim[n] = ok ? len - qlen + qs[n] + 1 : 0x7fffffff;
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

  while (todo) {
    const float vs_l = fmaxf(scale_l.y, kMinScale);
    const float kc_l = scale_l.x * r.scale_log2, lv_l = __log2f(vs_l), iv_l = 1.f / vs_l;
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
    next_units();
  }
  // ---- the unfinished block, by the wave whose turn it is
  if (rest && u1 == units && (nlist - u0) % kWaves == wave) {
    const uint16_t* kt = tail_ptr(st, false, bh, nfull) + c16 * kD + 16 * g;
    const uint16_t* vt = tail_ptr(st, true, bh, nfull) + c16 * kBlk + 16 * g;
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
    // a row by kThr / 16 lanes, 4 dims each at a time
    constexpr int kLanes = kThr / 16, kPieces = kD / 4 / kLanes;
    const int row = tid / kLanes, d = 4 * (tid % kLanes);
    const int col = col0 + 16 * n + row;
    if (col < r.cols) {
      float M = s_m[0][16 * n + row];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) M = fmaxf(M, s_m[w][16 * n + row]);
      const float mu = M == -INFINITY ? 0.f : M;
      f32x4 acc[kPieces];
#pragma unroll
      for (int k = 0; k < kPieces; ++k) acc[k] = f32x4{0.f, 0.f, 0.f, 0.f};
      float L = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float a = exp2_(s_m[w][16 * n + row] - mu);
        L += a * s_l[w][16 * n + row];
#pragma unroll
        for (int k = 0; k < kPieces; ++k) acc[k] += a * *reinterpret_cast<const f32x4*>(&s_o[w][row][4 * kLanes * k + d]);
      }
      const bool row_ok = col / r.G < qlen;
      const bool some = row_ok && L != 0.f;  // no such row, or no token: zeros
      const float inv = some ? 1.f / L : 0.f;
      const int64_t at = ((bh * r.cols + col) * P.splits + blockIdx.x);
#pragma unroll
      for (int k = 0; k < kPieces; ++k) {
        if (P.splits == 1)
          store_row<DT>(r, b, h, col, 4 * kLanes * k + d, some ? acc[k] * inv : f32x4{0.f, 0.f, 0.f, 0.f});
        else
          *reinterpret_cast<f32x4*>(P.part_o + at * kD + 4 * kLanes * k + d) = acc[k];
      }
      if (P.splits > 1 && tid % kLanes == 0)
        *reinterpret_cast<float2*>(P.part_ml + 2 * at) = row_ok ? part_record(M, L) : part_record(-INFINITY, 0.f);
    }
  }
}

struct CombineArgs {
  Rows r;
  const float* part_o;
  const float* part_ml;
  int64_t rows;
  int Hkv, splits;
};

// A row by PARTS groups of 32 lanes, each every PARTS-th split, 4 dims a lane; a workgroup has 8 / PARTS rows.  A split
// without a token for the row has offset -inf (and wrote no sums).  Bound by latency for few rows (8 groups: every load of
// up to 64 splits is asked for before the first is used), by memory for many.
template <int DT, int PARTS>
__global__ __launch_bounds__(kThr) void combine_kernel(CombineArgs P) {
  __shared__ __align__(16) float s_o[PARTS][kD];
  __shared__ float s_ml[PARTS][2];
  const Rows& r = P.r;
  const int tid = threadIdx.x, d = 4 * (tid & 31), part = (tid >> 5) % PARTS;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (8 / PARTS) + (tid >> 5) / PARTS;  // ((sequence, kv head), column)
  if (row >= P.rows) return;  // (PARTS 8: never)
  const int n = P.splits;
  const float* ml = P.part_ml + row * n * 2;
  const float* po = P.part_o + row * n * kD + d;
  float M = -INFINITY, L = 0.f;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int i0 = part; i0 < n; i0 += 8 * PARTS) {
    float2 x[8];
    f32x4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = i0 + k * PARTS;
      x[k] = float2{-INFINITY, 0.f};
      if (i < n) {
        x[k] = *reinterpret_cast<const float2*>(ml + 2 * i);
        v[k] = *reinterpret_cast<const f32x4*>(po + static_cast<int64_t>(i) * kD);
      }
    }
    float mx = M;
#pragma unroll
    for (int k = 0; k < 8; ++k) mx = fmaxf(mx, x[k].x);
    if (mx == -INFINITY) continue;
    const float a = exp2_(M - mx);
    M = mx;
    L *= a;
    acc *= a;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (x[k].x != -INFINITY) {
        const float w = exp2_(x[k].x - M);
        L = fmaf(w, x[k].y, L);
        acc += w * v[k];
      }
  }
  if constexpr (PARTS > 1) {
    *reinterpret_cast<f32x4*>(&s_o[part][d]) = acc;
    if ((tid & 31) == 0) {
      s_ml[part][0] = M;
      s_ml[part][1] = L;
    }
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int p = 1; p < PARTS; ++p) M = fmaxf(M, s_ml[p][0]);
    L = 0.f;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
      if (s_ml[p][0] != -INFINITY) {
        const float w = exp2_(s_ml[p][0] - M);
        L = fmaf(w, s_ml[p][1], L);
        acc += w * *reinterpret_cast<const f32x4*>(&s_o[p][d]);
      }
  }
  const float inv = L != 0.f ? 1.f / L : 0.f;
  if (L == 0.f) acc = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t bh = row / r.cols;
  store_row<DT>(r, static_cast<int>(bh / P.Hkv), static_cast<int>(bh % P.Hkv), static_cast<int>(row - bh * r.cols), d,
                acc * inv);
}

// --------------------------------------------------------------------------------------------------- block selection
constexpr int kSelThr = 512;
constexpr int kSelWaves = kSelThr / 64;
constexpr int kLdsKeys = 8192;     // so many keys of a (sequence, kv head) stay in LDS, more are read again from memory
// Up to so many finished blocks are chosen by counting, not by radix passes: a call over 20 blocks 4.7 us (by passes 6.8),
// over 128 6.0 (7.6), over 256 8.7 (8.1).
constexpr int kRankBlocks = kSelThr / 4;
constexpr uint32_t kForcedKey = 0xfffffffeu;  // above every score's
// Up to so many blocks (of max_len) one workgroup scores and selects, beyond that the scores are a launch of their own.  A
// selection in a replayed graph, one launch against two: 300 blocks 8.6 and 8.6 us (16 sequences 8.9 and 9.9), 400 9.1 and
// 8.4 (9.4, 9.9), 512 9.8 and 8.5 (10.4, 10.0), 640 11.8 and 9.3 (12.2, 11.8), 2048 23.0 and 10.3 (24.6, 20.8); a call outside a
// graph pays 2.5 us for the second launch.
constexpr int kFusedBlocks = 512;

struct SelectArgs {
  Store st;
  const void* q;
  int64_t q_sb, q_sh;
  const int* lens;
  int G, n, sink, recent;
  int max_len, max_blocks;  // bounds on the length and on the finished blocks
  uint32_t* keys;           // [B][Hkv][max_blocks], or null: scored by the selecting workgroup
  int* index;               // [B][Hkv][n]
};

// Order-preserving bits of a score (-0 made +0 before); larger is larger.
__device__ __forceinline__ uint32_t sort_bits(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

typedef int i32x4 __attribute__((ext_vector_type(4)));

// 16 of a kv head's queries in 8 bits: min(q8, 0) and max(q8, 0) of every dim, and their scales.
// By 512 threads: thread: query h0 + tid / 32, dims 4 (tid % 32) ..; into LDS, from where a wave reads its operands.
struct QueryCodes {
  uint32_t code[16][2][kD / 4];  // min(q8, 0), max(q8, 0)
  float scale[16];
};
template <int DT>
__device__ __forceinline__ void query_codes(const float (&x)[4], bool ok, QueryCodes& s, int tid) {
  float y[4], amax = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    y[j] = ok ? clamp_kv(x[j]) : 0.f;
    if constexpr (DT != LKV_DTYPE_F16) y[j] = h2f(f2h(y[j]));
    amax = fmaxf(amax, fabsf(y[j]));
  }
  amax = row16_max(amax);
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(amax), __float_as_uint(amax), false, false);
  amax = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const float inv = code_factor(amax);
  uint32_t un[4], up[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // rint by 1.5 * 2^23: the sum's low byte is the code
    const float t = y[j] * inv;
    un[j] = __float_as_uint(fminf(t, 0.f) + 12582912.f);
    up[j] = __float_as_uint(fmaxf(t, 0.f) + 12582912.f);
  }
  auto bytes = [](const uint32_t (&u)[4]) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400u),
                                 __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), 0x05040100u);
  };
  const int hh = (tid >> 5) & 15, d4 = tid & 31;
  s.code[hh][0][d4] = bytes(un);
  s.code[hh][1][d4] = bytes(up);
  if (d4 == 0) s.scale[hh] = amax * kStep;
}
template <int DT>
__device__ __forceinline__ void load_query4(const SelectArgs& P, int b, int h, int h0, int tid, float (&x)[4]) {
  const int64_t at = b * P.q_sb + static_cast<int64_t>(h * P.G + min(h0 + ((tid >> 5) & 15), P.G - 1)) * P.q_sh + 4 * (tid & 31);
  if constexpr (DT == LKV_DTYPE_F32) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(P.q) + at);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(P.q) + at);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = j < 2 ? v.x : v.y, u = (j & 1) ? w >> 16 : w & 0xffffu;
      x[j] = DT == LKV_DTYPE_F16 ? h2f(static_cast<uint16_t>(u)) : bf2f(u);
    }
  }
}
// Operands: column c16 = query, k slots = 16 bytes at dim 64 ks + 16 g.
__device__ __forceinline__ void query_operands(const QueryCodes& s, int c16, int g, i32x4 (&neg)[2], i32x4 (&pos)[2],
                                               float& qs) {
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    neg[ks] = *reinterpret_cast<const i32x4*>(&s.code[c16][0][16 * ks + 4 * g]);
    pos[ks] = *reinterpret_cast<const i32x4*>(&s.code[c16][1][16 * ks + 4 * g]);
  }
  qs = s.scale[c16];
}

// The lane's block row of a 16-block group: lowest codes, then highest ones.
__device__ __forceinline__ void load_ranges(const int8_t* p, i32x4 (&a)[4]) {
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) a[ks] = *reinterpret_cast<const i32x4*>(p + 64 * ks);
}

// Largest scaled product of the 16 columns with blocks 4 g + i of the group: the lane with c16 = i % 4 gets block i's.
__device__ __forceinline__ float group_best(const i32x4 (&a)[4], const i32x4 (&neg)[2], const i32x4 (&pos)[2], float qs,
                                            bool ok, int c16) {
  i32x4 d = i32x4{0, 0, 0, 0};
  d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[0], neg[0], d, 0, 0, 0);
  d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[1], neg[1], d, 0, 0, 0);
  d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[2], pos[0], d, 0, 0, 0);
  d = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[3], pos[1], d, 0, 0, 0);
  float best[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) best[i] = row16_max(ok ? static_cast<float>(d[i]) * qs : -INFINITY);
  return (c16 & 2) ? ((c16 & 1) ? best[3] : best[2]) : ((c16 & 1) ? best[1] : best[0]);
}

// Keys of 16 blocks per wave, for contexts whose scores are worth more than one workgroup per (sequence, kv head).
template <int DT>
__global__ __launch_bounds__(kSelThr) void score_kernel(SelectArgs P) {
  __shared__ __align__(16) QueryCodes s_q;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const int h = blockIdx.y, b = blockIdx.z;
  const Store& st = P.st;
  float x[4];
  load_query4<DT>(P, b, h, 0, tid, x);
  const int nfull = held_tokens(P.lens[b], P.max_len) / kBlk;
  const int64_t bh = static_cast<int64_t>(b) * st.Hkv + h;
  const int j0 = (blockIdx.x * kSelWaves + wave) * 16;
  if (static_cast<int>(blockIdx.x) * kSelWaves * 16 >= nfull) return;  // (the whole workgroup)
  i32x4 a[4];
  load_ranges(st.ranges + (bh * st.blocks + min(j0 + c16, nfull - 1)) * 2 * kD + 16 * g, a);
  const int j = j0 + 4 * g + (c16 & 3);
  const float ks = st.scales[2 * (bh * st.blocks + min(j, nfull - 1))];
  float best = -INFINITY;
  for (int h0 = 0; h0 < P.G; h0 += 16) {
    if (h0) {
      load_query4<DT>(P, b, h, h0, tid, x);
      __syncthreads();
    }
    query_codes<DT>(x, h0 + (tid >> 5) < P.G, s_q, tid);
    __syncthreads();
    i32x4 neg[2], pos[2];
    float qs;
    query_operands(s_q, c16, g, neg, pos, qs);
    best = fmaxf(best, group_best(a, neg, pos, qs, h0 + c16 < P.G, c16));
  }
  if (c16 < 4 && j < nfull) P.keys[bh * P.max_blocks + j] = sort_bits(best * ks);
}

// Over the wave: or, and, and the sum of the lanes up to this one (DPP, no LDS round trips).
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_or(uint32_t v) {
  v |= dpp_u<0xB1>(v);
  v |= dpp_u<0x4E>(v);
  v |= dpp_u<0x141>(v);
  v |= dpp_u<0x140>(v);
  return static_cast<uint32_t>(lane_i(v, 0) | lane_i(v, 16) | lane_i(v, 32) | lane_i(v, 48));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v += dpp_u<0x111>(v);  // row_shr:1, 2, 4, 8 (lanes shifted in from outside a row add 0)
  v += dpp_u<0x112>(v);
  v += dpp_u<0x114>(v);
  v += dpp_u<0x118>(v);
  const uint32_t r0 = lane_i(v, 15), r1 = lane_i(v, 31), r2 = lane_i(v, 47);
  const int row = (threadIdx.x & 63) >> 4;
  return v + (row > 0 ? r0 : 0u) + (row > 1 ? r1 : 0u) + (row > 2 ? r2 : 0u);
}

// The n highest keys of a (sequence, kv head), equal ones by index, as ascending indices; the rest of the row is -1.
// With P.keys null the workgroup computes them itself (every wave 16 blocks at a time, into LDS).  Bound by latency: one
// barrier a radix pass (a histogram each, every wave finds the bin by itself).
template <int DT>
__global__ __launch_bounds__(kSelThr) void select_kernel(SelectArgs P) {
  __shared__ __align__(16) uint32_t s_key[kLdsKeys];
  __shared__ __align__(16) uint32_t s_hist[4][256];
  __shared__ uint32_t s_or[kSelWaves], s_nor[kSelWaves];
  constexpr int kReg = 4;  // keys of a thread in registers: j = tid + kSelThr i
  __shared__ __align__(16) int s_cnt[kReg][2][kSelWaves];
  __shared__ __align__(16) QueryCodes s_q;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.x, b = blockIdx.y;
  const Store& st = P.st;
  float x[4];
  if (!P.keys) load_query4<DT>(P, b, h, 0, tid, x);  // (beside the length)
  const int nfull = held_tokens(P.lens[b], P.max_len) / kBlk;
  const int64_t bh = static_cast<int64_t>(b) * st.Hkv + h;
  int* out = P.index + bh * P.n;
  if (nfull <= P.n) {  // all of them
    for (int j = tid; j < P.n; j += kSelThr) out[j] = j < nfull ? j : -1;
    return;
  }
  const bool by_rank = nfull <= kRankBlocks;
  if (by_rank) {
    if (tid < 3) s_key[nfull + tid] = 0;  // (below every score's)
  } else {
    for (int i = tid; i < 4 * 256; i += kSelThr) s_hist[0][i] = 0;
  }
  // the first `sink` and the last `recent` blocks are in anyway: the others compete for the remaining places
  const int lo = min(P.sink, nfull), hi = max(nfull - P.recent, lo);  // [lo, hi) compete
  if (!P.keys) {
    const int c16 = lane & 15, g = lane >> 4;
    const int8_t* ranges = st.ranges + bh * st.blocks * 2 * kD + 16 * g;
    const float* scales = st.scales + 2 * bh * st.blocks;
    constexpr int kUn = 4;
    i32x4 a[kUn][4];
    float ks[kUn];
    auto load_groups = [&](int j0) {
#pragma unroll
      for (int u = 0; u < kUn; ++u) {
        const int jg = j0 + 16 * kSelWaves * u;
        load_ranges(ranges + static_cast<int64_t>(min(jg + c16, nfull - 1)) * 2 * kD, a[u]);
        ks[u] = scales[2 * min(jg + 4 * g + (c16 & 3), nfull - 1)];
      }
    };
    load_groups(16 * wave);  // (on their way beside the queries' codes)
    for (int h0 = 0; h0 < P.G; h0 += 16) {
      if (h0) {
        load_query4<DT>(P, b, h, h0, tid, x);
        __syncthreads();
      }
      query_codes<DT>(x, h0 + (tid >> 5) < P.G, s_q, tid);
      __syncthreads();
      i32x4 neg[2], pos[2];
      float qs;
      query_operands(s_q, c16, g, neg, pos, qs);
      const bool ok = h0 + c16 < P.G, end = h0 + 16 >= P.G;
      for (int j0 = 16 * wave; j0 < nfull;) {
        const int now = j0;
        float best[kUn], kn[kUn];
#pragma unroll
        for (int u = 0; u < kUn; ++u) {
          best[u] = group_best(a[u], neg, pos, qs, ok, c16);
          kn[u] = ks[u];
        }
        j0 += 16 * kSelWaves * kUn;
        if (j0 < nfull || !end) load_groups(j0 < nfull ? j0 : 16 * wave);
#pragma unroll
        for (int u = 0; u < kUn; ++u) {
          const int j = now + 16 * kSelWaves * u + 4 * g + (c16 & 3);
          if (c16 < 4 && j < nfull) {  // (a lane writes and reads back its own)
            if (h0) best[u] = fmaxf(best[u], __uint_as_float(s_key[j]));
            s_key[j] = !end                ? __float_as_uint(best[u])
                       : j >= lo && j < hi ? sort_bits(best[u] * kn[u])
                                           : kForcedKey;
          }
        }
      }
    }
  }
  const uint32_t* keys = P.keys ? P.keys + bh * P.max_blocks : nullptr;
  const bool in_lds = nfull <= kLdsKeys;
  if (keys && in_lds)
    for (int j = tid; j < nfull; j += kSelThr) s_key[j] = j >= lo && j < hi ? keys[j] : kForcedKey;
  __syncthreads();  // (keys and cleared histograms)
  if (by_rank) {
    // The number of blocks before block j in the order (key, index): four neighbouring threads a block count the keys
    // above its own, or equal to it at a lower index (four keys at a time: key > own - 1 before j's four, key > own from
    // there on, and j's own four once more for equal ones).
    const int j = tid >> 2, seg = tid & 3, mine = (j & ~3) + seg;
    const uint32_t own = s_key[min(j, nfull - 1)];
    uint32_t rank = mine < j && mine < nfull && s_key[mine] == own ? 1u : 0u;
    for (int c = 4 * seg; c < nfull; c += 16) {
      const u32x4 k = *reinterpret_cast<const u32x4*>(s_key + c);
      const uint32_t t = own - (c + 3 < j ? 1u : 0u);
      rank += (k[0] > t ? 1u : 0u) + (k[1] > t ? 1u : 0u) + (k[2] > t ? 1u : 0u) + (k[3] > t ? 1u : 0u);
    }
    rank += dpp_u<0xB1>(rank);
    rank += dpp_u<0x4E>(rank);
    const bool in = seg == 0 && j < nfull && rank < static_cast<uint32_t>(P.n);
    const uint64_t mask = wave_ballot(in);
    if (lane == 0) s_cnt[0][0][wave] = __popcll(mask);
    __syncthreads();
    int to = lane_prefix(mask);
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) to += w < wave ? s_cnt[0][0][w] : 0;
    if (in) out[to] = j;
    return;
  }
  auto key_at = [&](int j) { return in_lds ? s_key[j] : keys[j]; };
  const bool in_reg = nfull <= kReg * kSelThr;
  uint32_t kr[kReg];
#pragma unroll
  for (int i = 0; i < kReg; ++i) kr[i] = in_reg && tid + kSelThr * i < nfull ? s_key[tid + kSelThr * i] : 0u;
  int need = P.n - (nfull - (hi - lo));
  // f(key) for the thread's keys that compete
  auto each_key = [&](auto f) {
    if (in_reg) {
#pragma unroll
      for (int i = 0; i < kReg; ++i)
        if (tid + kSelThr * i >= lo && tid + kSelThr * i < hi) f(kr[i]);
    } else {
      for (int j = tid; j < hi; j += kSelThr)
        if (j >= lo) f(key_at(j));
    }
  };
  // bits in which the competing keys differ
  uint32_t any = 0, none = 0;  // set in some key, clear in some key
  each_key([&](uint32_t k) {
    any |= k;
    none |= ~k;
  });
  any = wave_or(any);
  none = wave_or(none);
  if (lane == 0) {
    s_or[wave] = any;
    s_nor[wave] = none;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) {
    any |= s_or[w];
    none |= s_nor[w];
  }
  any = __builtin_amdgcn_readfirstlane(any);
  const uint32_t diff = __builtin_amdgcn_readfirstlane(any & none);
  // radix selection from the highest of them down, 8 bits a pass (scores lie close: from the top of the word the first
  // pass would put nearly every key into one bin): the key of rank `need` is (prefix, lower bits)
  uint32_t prefix = need > 0 ? any : 0xffffffffu;  // (no place left: no key is above it)
  int top = diff ? 31 - __builtin_clz(diff) : -1;
  if (top >= 0 && need > 0) {
    prefix = top == 31 ? 0u : any & (0xffffffffu << (top + 1));
#pragma unroll 1
    for (int pass = 0; top >= 0; top -= 8, ++pass) {
      const int shift = max(top - 7, 0);
      const uint32_t mask = top == 31 ? 0u : 0xffffffffu << (top + 1), digit = (1u << (top - shift + 1)) - 1u;
      each_key([&](uint32_t k) {
        if ((k & mask) == prefix) atomicAdd(&s_hist[pass][(k >> shift) & digit], 1u);
      });
      __syncthreads();
      // lane: bins 4 lane .. + 3, and the counts above them
      const u32x4 c = *reinterpret_cast<const u32x4*>(&s_hist[pass][4 * lane]);
      const uint32_t sum = c[0] + c[1] + c[2] + c[3], upto = wave_scan(sum);
      uint32_t above = static_cast<uint32_t>(lane_i(static_cast<int>(upto), 63)) - upto;
      uint32_t bin = 0, over = 0;
      bool here = false;
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        if (above < static_cast<uint32_t>(need) && above + c[i] >= static_cast<uint32_t>(need)) {
          here = true;
          bin = 4 * lane + i;
          over = above;
        }
        above += c[i];
      }
      const int who = __builtin_ctzll(wave_ballot(here));  // (one lane)
      prefix |= static_cast<uint32_t>(lane_i(static_cast<int>(bin), who)) << shift;
      need -= lane_i(static_cast<int>(over), who);
    }
  }
  // the first and last blocks, the keys above `prefix` and the first `need` equal to it, in index order
  int base_gt = 0, base_eq = 0;
  // All counts at once and one barrier, where a round for each 512 keys would be three or more (2048 blocks 11.1 -> 10.2 us a
  // call; 1024 9.3 and 9.4, 512 9.7 and 10.2).
  if (in_reg && nfull > 2 * kSelThr) {
    uint64_t mg[kReg], me[kReg];
#pragma unroll
    for (int i = 0; i < kReg; ++i) {
      const int j = tid + kSelThr * i;
      const bool in = j >= lo && j < hi;
      mg[i] = wave_ballot(j < nfull && (!in || kr[i] > prefix));
      me[i] = wave_ballot(in && kr[i] == prefix);
      if (lane == 0) {
        s_cnt[i][0][wave] = __popcll(mg[i]);
        s_cnt[i][1][wave] = __popcll(me[i]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kReg; ++i) {
      int gt_before = base_gt + lane_prefix(mg[i]), eq_before = base_eq + lane_prefix(me[i]);
#pragma unroll
      for (int w = 0; w < kSelWaves; ++w) {
        const int cg = s_cnt[i][0][w], ce = s_cnt[i][1][w];
        if (w < wave) {
          gt_before += cg;
          eq_before += ce;
        }
        base_gt += cg;
        base_eq += ce;
      }
      if ((mg[i] >> lane & 1) || ((me[i] >> lane & 1) && eq_before < need))
        out[gt_before + min(eq_before, need)] = tid + kSelThr * i;
    }
    return;
  }
  for (int j0 = 0, it = 0; j0 < nfull; j0 += kSelThr, it ^= 1) {
    const int j = j0 + tid;
    const bool in = j >= lo && j < hi;
    const uint32_t k = in ? key_at(j) : 0u;
    const bool gt = j < nfull && (!in || k > prefix), eq = in && k == prefix;
    const uint64_t mg = wave_ballot(gt), me = wave_ballot(eq);
    if (lane == 0) {
      s_cnt[it][0][wave] = __popcll(mg);
      s_cnt[it][1][wave] = __popcll(me);
    }
    __syncthreads();  // (two sets of counts in turn: one barrier a round)
    int gt_before = base_gt + lane_prefix(mg), eq_before = base_eq + lane_prefix(me);
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) {
      const int cg = s_cnt[it][0][w], ce = s_cnt[it][1][w];
      if (w < wave) {
        gt_before += cg;
        eq_before += ce;
      }
      base_gt += cg;
      base_eq += ce;
    }
    if (gt || (eq && eq_before < need)) out[gt_before + min(eq_before, need)] = j;
  }
}

}  // namespace

Plan make_plan(int64_t B, int64_t Hkv, int64_t cols, int64_t units, bool listed) {
  Plan p;
  if (units < 1) units = 1;
  const int64_t cus = device_cu_count();
  p.nt = cols <= 16 ? 1 : cols <= 64 || listed ? 2 : 0;  // (the many-row kernel takes no list)
  const int64_t wide = p.nt ? 16 * p.nt : kManyCols;
  p.groups = static_cast<int>((cols + wide - 1) / wide);
  const int64_t items = B * Hkv * p.groups;
  // One workgroup a CU; two of the few-row kernel fit and would be no faster (32 sequences of up to 8192 tokens 68.2 us
  // with one, 70.1 with two a CU, 1 x 131072 tokens 52.5 and 53.4: more splits are more rows to join).
  const int64_t want = (cus + items - 1) / items;
  int64_t chunk = (units + want - 1) / want;
  if (p.nt)
    // a block for every wave; up to three for every wave are one split (512 tokens of one sequence 7.4 us, with rows to
    // join 9.1; 1024 tokens 10.0 and 9.1)
    chunk = units <= kOneSplit ? kOneSplit : (chunk + kWaves - 1) / kWaves * kWaves;
  else
    chunk = chunk < kManyChunk ? kManyChunk : chunk;
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

template <int DT>
void launch_combine(const CombineArgs& C, hipStream_t st) {
  // 8 rows a workgroup where that still gives every CU work
  if (C.rows >= 16ll * device_cu_count())
    hipLaunchKernelGGL((combine_kernel<DT, 1>), dim3(static_cast<unsigned>((C.rows + 7) / 8)), dim3(kThr), 0, st, C);
  else
    hipLaunchKernelGGL((combine_kernel<DT, 8>), dim3(static_cast<unsigned>(C.rows)), dim3(kThr), 0, st, C);
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
  return plan_bytes(make_plan(B, Hkv, cols, units_of(max_len, n_index), n_index > 0), B, Hkv, cols);
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
  const Plan p = make_plan(B, Hkv, cols, units_of(max_len, n_index), n_index > 0);
  LKV_REQUIRE(!p.nt || Hkv * p.groups < 65536, "kv8_attn: %lld query heads over a block list", (long long)Hq);
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
    const int64_t rows = B * Hkv * cols;
    const CombineArgs C{r, part_o, part_ml, rows, static_cast<int>(Hkv), p.splits};
    if (dtype == LKV_DTYPE_F32)
      launch_combine<LKV_DTYPE_F32>(C, st);
    else if (dtype == LKV_DTYPE_F16)
      launch_combine<LKV_DTYPE_F16>(C, st);
    else
      launch_combine<LKV_DTYPE_BF16>(C, st);
    LKV_LAUNCH_CHECK("kv8_attn combine");
  }
  return LKV_OK;
}

extern "C" size_t lkv_kv8_select_workspace_bytes(int64_t B, int64_t Hkv, int64_t max_len) {
  if (B <= 0 || Hkv <= 0 || max_len < 0 || max_len / kBlk <= kFusedBlocks) return 0;
  return static_cast<size_t>(B * Hkv * (max_len / kBlk)) * sizeof(uint32_t);
}

namespace {

template <int DT>
int launch_select(SelectArgs& P, int64_t B, hipStream_t st) {
  const unsigned Hkv = static_cast<unsigned>(P.st.Hkv);
  if (P.max_blocks > P.n && P.keys) {
    const int per = 16 * kSelWaves;
    hipLaunchKernelGGL(score_kernel<DT>, dim3(static_cast<unsigned>((P.max_blocks + per - 1) / per), Hkv,
                                              static_cast<unsigned>(B)), dim3(kSelThr), 0, st, P);
    LKV_LAUNCH_CHECK("kv8_select_blocks score");
  }
  hipLaunchKernelGGL(select_kernel<DT>, dim3(Hkv, static_cast<unsigned>(B)), dim3(kSelThr), 0, st, P);
  LKV_LAUNCH_CHECK("kv8_select_blocks");
  return LKV_OK;
}

}  // namespace

extern "C" int lkv_kv8_select_blocks(const lkv_kv8_store* store, const void* q, const int64_t* q_strides, int dtype,
                                     int64_t Hq, const int32_t* lens, int64_t max_len, int64_t n, int64_t sink,
                                     int64_t recent, int32_t* index, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  if (int rc = check_attn(store, Hq, 1, max_len, "kv8_select_blocks")) return rc;
  LKV_REQUIRE(dtype == LKV_DTYPE_F32 || dtype == LKV_DTYPE_F16 || dtype == LKV_DTYPE_BF16,
              "kv8_select_blocks: dtype %d", dtype);
  LKV_REQUIRE(n >= 1 && n < (1ll << 24) && sink >= 0 && recent >= 0 && sink <= n && recent <= n - sink,
              "kv8_select_blocks: %lld blocks with the first %lld and the last %lld among them", (long long)n,
              (long long)sink, (long long)recent);
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
  P.max_len = static_cast<int>(max_len);
  P.max_blocks = static_cast<int>(max_len / kBlk);
  P.keys = need ? static_cast<uint32_t*>(workspace) : nullptr;
  P.index = index;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == LKV_DTYPE_F32   ? launch_select<LKV_DTYPE_F32>(P, B, st)
         : dtype == LKV_DTYPE_F16 ? launch_select<LKV_DTYPE_F16>(P, B, st)
                                  : launch_select<LKV_DTYPE_BF16>(P, B, st);
}

extern "C" size_t lkv_kv8_sparse_attn_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t max_len, int64_t n) {
  const size_t a = lkv_kv8_select_workspace_bytes(B, Hkv, max_len);
  const size_t c = lkv_kv8_attn_workspace_bytes(B, Hq, Hkv, 1, max_len, n);
  return a > c ? a : c;
}

extern "C" int lkv_kv8_sparse_attn(const lkv_kv8_store* store, const void* q, const int64_t* q_strides, int dtype,
                                   int64_t Hq, const int32_t* lens, int64_t max_len, int64_t n, int64_t sink,
                                   int64_t recent, float scale, int32_t* index, void* out, const int64_t* out_strides,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  // (the scores are done with before the attention writes its partial sums: one workspace)
  if (int rc = check_attn(store, Hq, 1, max_len, "kv8_sparse_attn")) return rc;
  LKV_REQUIRE(store->batch == 0 || out, "kv8_sparse_attn: null pointer");
  if (store->batch)
    if (int rc = check_rows(out, out_strides, dtype, "kv8_sparse_attn", "out")) return rc;
  const size_t need = lkv_kv8_sparse_attn_workspace_bytes(store->batch, Hq, store->kv_heads, max_len, n);
  LKV_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
              "kv8_sparse_attn: workspace of %zu bytes (16-byte aligned) required, got %zu", need, workspace_bytes);
  if (int rc = lkv_kv8_select_blocks(store, q, q_strides, dtype, Hq, lens, max_len, n, sink, recent, index, workspace,
                                     workspace_bytes, stream))
    return rc;
  return lkv_kv8_attn(store, q, q_strides, dtype, Hq, 1, lens, nullptr, max_len, index, n, scale, out, out_strides,
                      workspace, workspace_bytes, stream);
}
