// Attention of one query per sequence over the 16-bit paged KV cache (lkv_pages_decode_attn), and the join of partial sums.
//
//   split kernel  grid (splits, kv heads x column tiles, sequences), 4 waves.  A wave takes every 4th chunk of 32 tokens of
//                 its split, each row read once and straight into registers, and runs on v_mfma_f32_16x16x32
//                   scores^T (16 tokens x 16 columns)  A = 16 rows of keys, B = the columns' queries,
//                   softmax per lane (its column, 8 of the chunk's tokens), running offset in the log2 domain,
//                   out^T   (16 dims x 16 columns) += A = 16 dims of 32 rows of values (paired by v_perm), B = the weights.
//   join          combines the splits' (offset, sum, row) in fp32.
//
// A product has 16 columns and a sequence fills Hq / Hkv of them.  The others are given to its neighbours: of the
// 16 / (Hq / Hkv) sequences of an aligned group, those whose pages in this split are the same (forked from one prompt) and
// end at the same token are the columns of one workgroup, that of the first of them; the workgroups of the others end at
// once.  Pages are compared where they are staged, so sharing needs no plan and no call of its own.
#include "pages_common.h"

namespace lkv {
namespace pages {
namespace {

constexpr int kThr = 256;
constexpr int kWaves = 4;
constexpr int kChunk = 32;
constexpr int kStep = kChunk * kWaves;  // tokens of a workgroup's step
constexpr int kMaxPages = 1024;         // page ids of a split, staged in LDS
constexpr int kMaxSplits = 1024;

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

struct DecodeArgs {
  Pages st;
  const uint16_t* kv;  // the layer's pages
  const uint16_t* q;
  int64_t q_ss, q_sh;
  uint16_t* out;
  int64_t o_ss, o_sh;
  int Hq, G;
  int tiles;    // column tiles of a kv head: 1, or ceil(G / 16)
  int group;    // sequences of a group: 16 / G, at least 1
  int max_len, chunk, splits;  // tokens of a split
  float scale_log2;
  float* part_o;   // [seqs * Hq][splits][128]
  float* part_ml;  // [seqs * Hq][splits][2]
};

template <int DT>
__global__ __launch_bounds__(kThr, 2) void split_kernel(DecodeArgs P) {
  constexpr int kRow = kD + 4;  // floats of a staged row
  __shared__ __align__(16) float s_o[kWaves][16][kRow];
  __shared__ float s_m[kWaves][16], s_l[kWaves][16];
  __shared__ int s_page[kMaxPages];
  __shared__ int s_other;  // sequences of the group that read other pages
  const Pages& st = P.st;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const int split = blockIdx.x, h = blockIdx.y / P.tiles, tile = blockIdx.y - h * P.tiles, s = blockIdx.z;
  const int G = P.G;

  const int len = min(held(st, st.lens[s]), P.max_len);
  const int t0 = split * P.chunk, t1 = min(t0 + P.chunk, len);
  // columns of the workgroup's own sequence: heads 16 tile .. of its kv head
  const int own_heads = min(G - 16 * tile, 16);
  if (t0 >= t1) {  // uniform: nothing here
    if (P.splits == 1) {
      for (int e = tid; e < own_heads * (kD / 8); e += kThr)
        *reinterpret_cast<u32x4*>(P.out + s * P.o_ss + (static_cast<int64_t>(h) * G + 16 * tile + e / (kD / 8)) * P.o_sh +
                                  8 * (e % (kD / 8))) = u32x4{};
    } else if (tid < own_heads) {
      const int64_t row = static_cast<int64_t>(s) * P.Hq + h * G + 16 * tile + tid;
      *reinterpret_cast<float2*>(P.part_ml + 2 * (row * P.splits + split)) = part_record(-INFINITY, 0.f);
    }
    return;
  }

  // ---- the split's pages, and who else reads them
  const int base = s - s % P.group;
  const int members = min(P.group, st.seqs - base);
  const int page0 = t0 >> st.lg, pages = ((t1 - 1) >> st.lg) - page0 + 1;
  int mine = 1 << (s - base);  // members in this workgroup, as bits
  if (P.group > 1) {
    if (tid == 0) s_other = 0;
    __syncthreads();
  }
  {
    const int* row = st.table + static_cast<int64_t>(s) * st.width + page0;
    int other = 0;
    for (int i = tid; i < pages; i += kThr) {
      const int p = page_id(st, row[i]);
      s_page[i] = p;
      for (int j = 0; j < members; ++j) {
        const int q = page_id(st, st.table[static_cast<int64_t>(base + j) * st.width + page0 + i]);
        other |= q != p ? 1 << j : 0;
      }
    }
    if (P.group > 1) {
      if (tid < members && min(t0 + P.chunk, min(held(st, st.lens[base + tid]), P.max_len)) != t1) other |= 1 << tid;
      if (other) atomicOr(&s_other, other);
    }
  }
  __syncthreads();
  if (P.group > 1) {
    mine = ~__builtin_amdgcn_readfirstlane(s_other) & ((1 << members) - 1);
    if (mine & ((1 << (s - base)) - 1)) return;  // uniform: an earlier sequence's workgroup does it
  }

  // ---- the lane's column: head `head` of sequence `seq`
  const int slot = P.group > 1 ? c16 / G : 0;
  const bool ok = P.group > 1 ? slot < members && ((mine >> slot) & 1) : c16 < own_heads;
  const int seq = P.group > 1 ? base + min(slot, members - 1) : s;
  const int head = h * G + (P.group > 1 ? c16 - slot * G : 16 * tile + min(c16, own_heads - 1));
  u32x4 qf[4];  // dims 32 kb + 8 g ..
  {
    const uint16_t* p = P.q + seq * P.q_ss + head * P.q_sh + 8 * g;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) qf[kb] = ok ? *reinterpret_cast<const u32x4*>(p + 32 * kb) : u32x4{};
  }

  // ---- chunks c = t0 + 32 (wave + 4 i): keys of tokens c + 16 tt + lane % 16, values j of tokens
  // c + 16 (j / 4) + 4 (lane / 16) + j % 4; tokens past the end read the last one, masked below
  const int64_t run = run_numbers(st);
  const int mask = page_size(st) - 1;
  auto at = [&](int t) {  // a token's row of keys in the layer
    t = min(t, t1 - 1);
    return s_page[(t >> st.lg) - page0] * (2 * st.H * run) + h * run + (t & mask) * kD;
  };
  u32x4 kr[2][4], vr[8];
  auto load_chunk = [&](int c) {
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const uint16_t* p = P.kv + at(c + 16 * tt + c16) + 8 * g;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) kr[tt][kb] = *reinterpret_cast<const u32x4*>(p + 32 * kb);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      vr[j] = *reinterpret_cast<const u32x4*>(P.kv + at(c + 16 * (j >> 2) + 4 * g + (j & 3)) + st.H * run + 8 * c16);
  };
  float m = -INFINITY, l = 0.f;
  f32x4 o[8];  // o[t] row 4 g + i: dim 8 (4 g + i) + t of the lane's column
#pragma unroll
  for (int t = 0; t < 8; ++t) o[t] = f32x4{};
  int c = t0 + kChunk * wave;
  if (c < t1) load_chunk(c);
  for (; c < t1; c += kStep) {
    f32x4 sc[2];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      sc[tt] = f32x4{};
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) sc[tt] = mfma16<DT>(kr[tt][kb], qf[kb], sc[tt]);
    }
    float x[8], mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = sc[e >> 2][e & 3] * P.scale_log2;
    if (c + kChunk > t1) {  // uniform: the last tokens.  Rows past them are no numbers of this sequence
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool past = c + 16 * (e >> 2) + 4 * g + (e & 3) >= t1;
        x[e] = past ? -INFINITY : x[e];
        if (past) vr[e] = u32x4{};
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) mx = fmaxf(mx, x[e]);
    if (wave_ballot(mx - m > kMaxWeight || m == -INFINITY)) {  // uniform: a new offset somewhere
      mx = groups_max(mx);
      const float mn = mx - m > kMaxWeight ? mx - kTopWeight : m;
      const float alpha = exp2_(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= alpha;
#pragma unroll
      for (int t = 0; t < 8; ++t) o[t] = o[t] * alpha;
    }
    const float mu = m == -INFINITY ? 0.f : m;
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = exp2_(x[e] - mu);
    const u32x4 pb = u32x4{pack<DT>(w[0], w[1]), pack<DT>(w[2], w[3]), pack<DT>(w[4], w[5]), pack<DT>(w[6], w[7])};
#pragma unroll
    for (int e = 0; e < 4; ++e) l = add_pair<DT>(pb[e], l);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      u32x4 a;
#pragma unroll
      for (int pp = 0; pp < 4; ++pp)
        a[pp] = __builtin_amdgcn_perm(vr[2 * pp + 1][t >> 1], vr[2 * pp][t >> 1], (t & 1) ? 0x07060302u : 0x05040100u);
      o[t] = mfma16<DT>(a, pb, o[t]);
    }
    if (c + kStep < t1) load_chunk(c + kStep);
  }

  // ---- the four waves' sums
  l = groups_sum(l);
  if (g == 0) {
    s_m[wave][c16] = l != l ? 0.f : m;
    s_l[wave][c16] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float* dst = &s_o[wave][c16][8 * (4 * g + i)];
    *reinterpret_cast<f32x4*>(dst) = f32x4{o[0][i], o[1][i], o[2][i], o[3][i]};
    *reinterpret_cast<f32x4*>(dst + 4) = f32x4{o[4][i], o[5][i], o[6][i], o[7][i]};
  }
  __syncthreads();
  const int col = tid >> 4, d = 8 * (tid & 15);
  const int cslot = P.group > 1 ? col / G : 0;
  const bool cok = P.group > 1 ? cslot < members && ((mine >> cslot) & 1) : col < own_heads;
  if (!cok) return;
  const int cseq = P.group > 1 ? base + cslot : s;
  const int64_t chead = h * G + (P.group > 1 ? col - cslot * G : 16 * tile + col);
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) M = fmaxf(M, s_m[w][col]);
  float L = 0.f, r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float mw = s_m[w][col];
    if (mw == -INFINITY) continue;  // no weight yet: its sums are zeros
    const float wt = exp2_(mw - M);
    L = fmaf(wt, s_l[w][col], L);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = fmaf(wt, s_o[w][col][d + i], r[i]);
  }
  if (P.splits == 1) {
    const float inv = L != 0.f ? 1.f / L : 0.f;
    *reinterpret_cast<u32x4*>(P.out + cseq * P.o_ss + chead * P.o_sh + d) =
        u32x4{pack<DT>(r[0] * inv, r[1] * inv), pack<DT>(r[2] * inv, r[3] * inv), pack<DT>(r[4] * inv, r[5] * inv),
              pack<DT>(r[6] * inv, r[7] * inv)};
    return;
  }
  const int64_t rec = (static_cast<int64_t>(cseq) * P.Hq + chead) * P.splits + split;
  if ((tid & 15) == 0) *reinterpret_cast<float2*>(P.part_ml + 2 * rec) = part_record(M, L);
  *reinterpret_cast<f32x4*>(P.part_o + rec * kD + d) = f32x4{r[0], r[1], r[2], r[3]};
  *reinterpret_cast<f32x4*>(P.part_o + rec * kD + d + 4) = f32x4{r[4], r[5], r[6], r[7]};
}

struct JoinArgs {
  const float* part_o;
  const float* part_ml;
  uint16_t* out;
  int64_t o_st, o_sh;
  const int* cu;
  int n;
  int rows, splits, heads;
};

// A group of 32 lanes sums splits of one row, 4 dims a lane.  ONE: the eight groups of a workgroup take a row each (few
// splits); otherwise they share one row, every eighth split each, and meet in LDS.
template <int DT, bool ONE>
__global__ __launch_bounds__(kThr) void join_kernel(JoinArgs A) {
  __shared__ __align__(16) float s_o[8][kD];
  __shared__ float s_l[8];
  const int tid = threadIdx.x, grp = tid >> 5, d = 4 * (tid & 31);
  const int row = ONE ? blockIdx.x * 8 + grp : blockIdx.x;
  if (row >= A.rows) return;  // (whole groups; with ONE no barrier follows)
  const int t = row / A.heads, head = row - t * A.heads;
  if (A.cu && (t < A.cu[0] || t >= A.cu[A.n])) return;
  const float2* ml = reinterpret_cast<const float2*>(A.part_ml) + static_cast<int64_t>(row) * A.splits;
  const float* po = A.part_o + static_cast<int64_t>(row) * A.splits * kD + d;
  float M = -INFINITY;
  for (int i = tid & 31; i < A.splits; i += 32) M = fmaxf(M, ml[i].x);
#pragma unroll
  for (int x = 16; x; x >>= 1) M = fmaxf(M, __shfl_xor(M, x));
  float L = 0.f;
  f32x4 o = f32x4{};
  for (int i = ONE ? 0 : grp; i < A.splits; i += ONE ? 1 : 8) {
    const float2 r = ml[i];
    if (r.x == -INFINITY) continue;  // an empty part: its row was not written
    const float w = exp2_(r.x - M);
    const f32x4 x = *reinterpret_cast<const f32x4*>(po + static_cast<int64_t>(i) * kD);
    L = fmaf(w, r.y, L);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = fmaf(w, x[k], o[k]);
  }
  if constexpr (!ONE) {
    *reinterpret_cast<f32x4*>(&s_o[grp][d]) = o;
    if ((tid & 31) == 0) s_l[grp] = L;
    __syncthreads();
    if (grp) return;
    o = f32x4{};
    L = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      o = o + *reinterpret_cast<const f32x4*>(&s_o[k][d]);
      L += s_l[k];
    }
  }
  const float inv = L != 0.f ? 1.f / L : 0.f;
  *reinterpret_cast<uint2*>(A.out + t * A.o_st + head * A.o_sh + d) =
      uint2{pack<DT>(o[0] * inv, o[1] * inv), pack<DT>(o[2] * inv, o[3] * inv)};
}

struct DecodePlan {
  int chunk, splits;
};

DecodePlan decode_plan(int64_t S, int64_t Hq, int64_t Hkv, int64_t max_len) {
  const int64_t tiles = (Hq / Hkv + 15) / 16, pairs = S * Hkv * tiles;
  const int64_t steps = (max_len + kStep - 1) / kStep;
  int64_t splits = 1;
  if (steps > 3) {
    const int64_t target = 4ll * device_cu_count();
    splits = (target + pairs - 1) / pairs;
    splits = splits < 1 ? 1 : splits;
    splits = splits > steps ? steps : splits;
    splits = splits > kMaxSplits ? kMaxSplits : splits;
  }
  int64_t chunk = (steps + splits - 1) / splits;
  // page ids of a split fit their place whatever the page size: 16 tokens a page and the one that it begins in
  const int64_t most = (kMaxPages - 1) * 16 / kStep;
  chunk = chunk > most ? most : (chunk < 1 ? 1 : chunk);
  DecodePlan p;
  p.splits = static_cast<int>(steps <= chunk ? 1 : (steps + chunk - 1) / chunk);
  p.chunk = static_cast<int>(chunk * kStep);
  return p;
}

}  // namespace

int launch_join(const float* part_o, const float* part_ml, int64_t rows, int64_t splits, int64_t heads, void* out,
                int64_t o_st, int64_t o_sh, int dtype, const int* cu, int n, hipStream_t stream, const char* what) {
  const JoinArgs A{part_o, part_ml, static_cast<uint16_t*>(out), o_st, o_sh, cu, n, static_cast<int>(rows),
                   static_cast<int>(splits), static_cast<int>(heads)};
  const bool one = splits <= 8;
  const dim3 grid(static_cast<unsigned>(one ? (rows + 7) / 8 : rows));
  if (dtype == LKV_DTYPE_F16) {
    if (one)
      hipLaunchKernelGGL((join_kernel<LKV_DTYPE_F16, true>), grid, dim3(kThr), 0, stream, A);
    else
      hipLaunchKernelGGL((join_kernel<LKV_DTYPE_F16, false>), grid, dim3(kThr), 0, stream, A);
  } else {
    if (one)
      hipLaunchKernelGGL((join_kernel<LKV_DTYPE_BF16, true>), grid, dim3(kThr), 0, stream, A);
    else
      hipLaunchKernelGGL((join_kernel<LKV_DTYPE_BF16, false>), grid, dim3(kThr), 0, stream, A);
  }
  LKV_LAUNCH_CHECK(what);
  return LKV_OK;
}

}  // namespace pages
}  // namespace lkv

using namespace lkv;
using namespace lkv::pages;

extern "C" size_t lkv_pages_decode_attn_workspace_bytes(int64_t seqs, int64_t Hq, int64_t Hkv, int64_t max_len) {
  if (seqs < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || max_len < 0) return 0;
  const DecodePlan p = decode_plan(seqs, Hq, Hkv, max_len);
  return p.splits == 1 ? 0 : static_cast<size_t>(seqs * Hq) * p.splits * (kD + 2) * 4;
}

extern "C" int lkv_pages_decode_attn(const lkv_pages* p, int64_t layer, const void* q, const int64_t* q_strides,
                                     int64_t Hq, int64_t max_len, float scale, void* out, const int64_t* out_strides,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "pages_decode_attn";
  if (int rc = check_pages(p, what)) return rc;
  LKV_REQUIRE(layer >= 0 && layer < p->layers, "%s: layer %lld of %lld", what, (long long)layer, (long long)p->layers);
  LKV_REQUIRE(Hq > 0 && Hq % p->kv_heads == 0 && Hq < (1 << 20), "%s: %lld query heads over %lld kv heads", what,
              (long long)Hq, (long long)p->kv_heads);
  LKV_REQUIRE(max_len >= 0 && max_len <= p->width * p->page_size, "%s: max_len=%lld outside sequences of up to %lld tokens",
              what, (long long)max_len, (long long)(p->width * p->page_size));
  if (int rc = check_rows(q, q_strides, what, "q")) return rc;
  if (int rc = check_rows(out, out_strides, what, "out")) return rc;
  const int64_t G = Hq / p->kv_heads, tiles = (G + 15) / 16;
  LKV_REQUIRE(p->kv_heads * tiles < 65536 && p->seqs * Hq < (1ll << 28), "%s: %lld query heads", what, (long long)Hq);
  const DecodePlan plan = decode_plan(p->seqs, Hq, p->kv_heads, max_len);
  const size_t need = lkv_pages_decode_attn_workspace_bytes(p->seqs, Hq, p->kv_heads, max_len);
  LKV_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
              "%s: a 16-byte aligned workspace of %zu bytes required, got %zu", what, need, workspace_bytes);
  DecodeArgs A{};
  A.st = device_pages(p);
  A.kv = A.st.pool + layer * p->pages * 2 * p->kv_heads * p->page_size * kD;
  A.q = static_cast<const uint16_t*>(q);
  A.q_ss = q_strides[0];
  A.q_sh = q_strides[1];
  A.out = static_cast<uint16_t*>(out);
  A.o_ss = out_strides[0];
  A.o_sh = out_strides[1];
  A.Hq = static_cast<int>(Hq);
  A.G = static_cast<int>(G);
  A.tiles = static_cast<int>(tiles);
  A.group = G <= 8 ? static_cast<int>(16 / G) : 1;
  A.max_len = static_cast<int>(max_len);
  A.chunk = plan.chunk;
  A.splits = plan.splits;
  A.scale_log2 = scale * kLog2e;
  A.part_o = static_cast<float*>(workspace);
  A.part_ml = A.part_o + static_cast<size_t>(p->seqs * Hq) * plan.splits * kD;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(plan.splits), static_cast<unsigned>(p->kv_heads * tiles),
                  static_cast<unsigned>(p->seqs));
  if (p->dtype == LKV_DTYPE_F16)
    hipLaunchKernelGGL(split_kernel<LKV_DTYPE_F16>, grid, dim3(kThr), 0, s, A);
  else
    hipLaunchKernelGGL(split_kernel<LKV_DTYPE_BF16>, grid, dim3(kThr), 0, s, A);
  LKV_LAUNCH_CHECK(what);
  if (plan.splits == 1) return LKV_OK;
  return launch_join(A.part_o, A.part_ml, p->seqs * Hq, plan.splits, Hq, out, A.o_ss, A.o_sh, p->dtype, nullptr, 0, s,
                     "pages_decode_attn join");
}
