// Attention of one query per sequence over the 16-bit paged KV cache (lkv_pages_decode_attn), of a few (lkv_pages_prefill_attn
// with up to 32 columns = queries x heads of a kv head), and the join of partial sums.
//
//   split kernel  grid (splits, kv heads x column tiles, sequences), 4 waves.  A wave takes every 4th chunk of 32 tokens of
//                 its split, each row read once and straight into registers, and runs on v_mfma_f32_16x16x32
//                   scores^T (16 tokens x 16 columns)  A = 16 rows of keys, B = the columns' queries,
//                   softmax per lane (its column, 8 of the chunk's tokens), running offset in the log2 domain,
//                   out^T   (16 dims x 16 columns) += A = 16 dims of 32 rows of values (paired by v_perm), B = the weights.
//   join          combines the splits' (offset, sum, row) in fp32.
//
// A product has 16 columns and a sequence fills Hq / Hkv of them.  The others, and those of a second product over the same
// rows, are given to its neighbours: of the 32 / (Hq / Hkv) sequences of an aligned group, those that begin the split on the
// same page (forked from one prompt) are read once as far as all of them name the same pages.  Their workgroups divide that
// part among themselves, each for the columns of all; what follows each reads for its own.  A split has a record for its own
// part and one for every sequence of the group.  Pages are compared where they are staged, so sharing needs no plan and no
// call of its own.
//
// A few newest queries of a sequence (drafted tokens, checked in one pass) are the columns of its workgroups in the same way;
// those that do not see the last tokens have weight 0 there.  Where such a token's value is no number, 0 times it is none
// either: it counts as 0 then, and a second product counts, of each kind, those that a column sees.
//
// Bound by memory: a wave's next chunk (16 KB) is on its way while it computes this one, 8 waves a CU (229 registers; 250 with
// masks), so that 128 KB a CU are.  32/8 heads, by card: 32 sequences of 8192 tokens 186 us, 5.8 TB/s; 32 of 1.6-8 K 135-136 us, 4.8
// TB/s (the longest end last); 131072 tokens of one sequence 98-99 us, of them 95 (5.7 TB/s) reading and 5 joining 64 splits; 32
// beams over 4 prompts of 8192 tokens, 152 MB read once, 34-40 us.  5 drafted tokens of 8 sequences of 4096 29-34 us, of them 26
// (5.1 TB/s) reading; in the prefill kernel, whose waves wait for each other's rows, 37 where it takes 29.
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
constexpr size_t kMostBytes = size_t{1} << 28;  // of records where the plan has the choice

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
  int g_small;  // c / G = c * g_small >> 16 for columns c of a group
  int tiles;    // column tiles of a kv head: 1, or ceil(G / 16)
  int group;    // sequences of a group: up to 32 / G, or 1 where none are shared
  int max_len, chunk, splits;  // tokens of a split
  int slots;    // records of a row: splits, or splits (group + 1): a split's own part, and the shared ones
  const int* cu;  // rows of several queries a sequence: where they begin
  int rows, fill;
  float scale_log2;
  float* part_o;   // [seqs * Hq][slots][128]
  float* part_ml;  // [seqs * Hq][slots][2]
};

constexpr int kRow = kD + 4;  // floats of a staged row
struct Staged {
  float o[kWaves][16][kRow];
  float m[kWaves][32], l[kWaves][32];
  int page[kMaxPages];
  int end[32], same[32], member[32];
};

// Attention over tokens [lo, hi) of the workgroup's split for `cols` columns, 16 NT at most; where(c, row, head) says which
// query column c is and slot where its record goes (no slots: the result itself).  Column c sees tokens below sees(c) (MASKED),
// all of them those below `free`.  pages(i): the i-th page id of the sequence's row from page0 on.
template <int DT, int NT, bool MASKED, class Where, class Sees, class PageOf>
__device__ __forceinline__ void attend(const DecodeArgs& P, Staged& sh, int h, int page0, int lo, int hi, int free, int cols,
                                       int slot, Where where, Sees sees, PageOf pages) {
  const Pages& st = P.st;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  u32x4 qf[NT][4];  // dims 32 kb + 8 g ..
  int lim[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {  // (a column past the last is the last once more)
    int row, head;
    where(min(16 * n + c16, cols - 1), row, head);
    const uint16_t* p = P.q + row * P.q_ss + head * P.q_sh + 8 * g;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) qf[n][kb] = *reinterpret_cast<const u32x4*>(p + 32 * kb);
    lim[n] = MASKED ? min(sees(min(16 * n + c16, cols - 1)), hi) : hi;
  }
  // ---- chunks c = lo + 32 (wave + 4 i): keys of tokens c + 16 tt + lane % 16, values j of tokens
  // c + 16 (j / 4) + 4 (lane / 16) + j % 4; tokens past the end read the last one, masked below
  const int64_t run = run_numbers(st);
  const int mask = page_size(st) - 1;
  auto at = [&](int t) {  // a token's row of keys in the layer
    t = min(t, hi - 1);
    return pages((t >> st.lg) - page0) * (2 * st.H * run) + h * run + (t & mask) * kD;
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
  float m[NT], l[NT];
  f32x4 o[NT][8];  // o[n][t] row 4 g + i: dim 8 (4 g + i) + t of the lane's column of tile n
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int t = 0; t < 8; ++t) o[n][t] = f32x4{};
  }
  int c = lo + kChunk * wave;
  if (c < hi) load_chunk(c);
#pragma unroll 1
  for (; c < hi; c += kStep) {
    const bool last = c + kChunk > free;  // uniform: rows past the end are no numbers of this sequence
    bool odd = false;                     // uniform: a value that not all columns see is no number
    if (last) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + 16 * (e >> 2) + 4 * g + (e & 3) >= hi) vr[e] = u32x4{};
      if constexpr (MASKED) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            any |= (vr[e][k] & 0x7fffu) >= inf_bits<DT>() || (vr[e][k] >> 16 & 0x7fffu) >= inf_bits<DT>();
        odd = wave_ballot(any) != 0;
      }
    }
    u32x4 pb[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4 sc[2];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        sc[tt] = f32x4{};
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) sc[tt] = mfma16<DT>(kr[tt][kb], qf[n][kb], sc[tt]);
      }
      float x[8], mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = sc[e >> 2][e & 3] * P.scale_log2;
      if (last) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = c + 16 * (e >> 2) + 4 * g + (e & 3) >= lim[n] ? -INFINITY : x[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, x[e]);
      if (wave_ballot(mx - m[n] > max_weight<DT>() || m[n] == -INFINITY)) {  // uniform: a new offset somewhere
        mx = groups_max(mx);
        const float mn = mx - m[n] > max_weight<DT>() ? mx - top_weight<DT>() : m[n];
        const float alpha = exp2_(m[n] - (mn == -INFINITY ? 0.f : mn));
        m[n] = mn;
        l[n] *= alpha;
#pragma unroll
        for (int t = 0; t < 8; ++t) o[n][t] = o[n][t] * alpha;
      }
      const float mu = m[n] == -INFINITY ? 0.f : m[n];
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = exp2_(x[e] - mu);
      pb[n] = u32x4{pack<DT>(w[0], w[1]), pack<DT>(w[2], w[3]), pack<DT>(w[4], w[5]), pack<DT>(w[6], w[7])};
#pragma unroll
      for (int e = 0; e < 4; ++e) l[n] = add_pair<DT>(pb[n][e], l[n]);
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      u32x4 a;
#pragma unroll
      for (int pp = 0; pp < 4; ++pp)
        a[pp] = __builtin_amdgcn_perm(vr[2 * pp + 1][t >> 1], vr[2 * pp][t >> 1], (t & 1) ? 0x07060302u : 0x05040100u);
      if constexpr (MASKED) {
        if (odd) {
          u32x4 fine, kind;
          no_numbers<DT>(a, fine, kind);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            u32x4 seen;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int t0 = c + 16 * (k >> 1) + 4 * g + 2 * (k & 1);  // its two tokens
              seen[k] = (t0 < lim[n] ? one_bits<DT>() : 0u) | (t0 + 1 < lim[n] ? one_bits<DT>() << 16 : 0u);
            }
            o[n][t] = mfma16<DT>(fine, pb[n], o[n][t]);
            const f32x4 count = mfma16<DT>(kind, seen, f32x4{});
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float sum = o[n][t][i];
              add_counted(count[i], sum);
              o[n][t][i] = sum;
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          continue;
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) o[n][t] = mfma16<DT>(a, pb[n], o[n][t]);
    }
    if (c + kStep < hi) load_chunk(c + kStep);
  }

  // ---- the four waves' sums, a column tile after the other
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float ln = groups_sum(l[n]);
    __syncthreads();  // (what lies there is read)
    if (g == 0) {
      sh.m[wave][c16] = ln != ln ? 0.f : m[n];
      sh.l[wave][c16] = ln;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float* dst = &sh.o[wave][c16][8 * (4 * g + i)];
      *reinterpret_cast<f32x4*>(dst) = f32x4{o[n][0][i], o[n][1][i], o[n][2][i], o[n][3][i]};
      *reinterpret_cast<f32x4*>(dst + 4) = f32x4{o[n][4][i], o[n][5][i], o[n][6][i], o[n][7][i]};
    }
    __syncthreads();
    int thread = tid;
    __asm__ volatile("" : "+v"(thread));  // (what follows from it is not kept through the chunks)
    const int col = thread >> 4, d = 8 * (thread & 15);
    if (16 * n + col >= cols) continue;
    int row, head;
    where(16 * n + col, row, head);
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, sh.m[w][col]);
    float L = 0.f, r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mw = sh.m[w][col];
      if (mw == -INFINITY) continue;  // no weight yet: its sums are zeros
      const float wt = exp2_(mw - M);
      L = fmaf(wt, sh.l[w][col], L);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = fmaf(wt, sh.o[w][col][d + i], r[i]);
    }
    if (P.slots == 1) {
      const float inv = L != 0.f ? 1.f / L : 0.f;
      *reinterpret_cast<u32x4*>(P.out + row * P.o_ss + head * P.o_sh + d) =
          u32x4{pack<DT>(r[0] * inv, r[1] * inv), pack<DT>(r[2] * inv, r[3] * inv), pack<DT>(r[4] * inv, r[5] * inv),
                pack<DT>(r[6] * inv, r[7] * inv)};
      continue;
    }
    const int64_t rec = (static_cast<int64_t>(row) * P.Hq + head) * P.slots + slot;
    if (d == 0) *reinterpret_cast<float2*>(P.part_ml + 2 * rec) = part_record(M, L);
    *reinterpret_cast<f32x4*>(P.part_o + rec * kD + d) = f32x4{r[0], r[1], r[2], r[3]};
    *reinterpret_cast<f32x4*>(P.part_o + rec * kD + d + 4) = f32x4{r[4], r[5], r[6], r[7]};
  }
}

template <int DT>
__global__ __launch_bounds__(kThr, 2) void split_kernel(DecodeArgs P) {
  __shared__ __align__(16) Staged sh;
  const Pages& st = P.st;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int split = blockIdx.x, h = blockIdx.y / P.tiles, tile = blockIdx.y - h * P.tiles, s = blockIdx.z;
  const int G = P.G;

  const int len = min(held(st, st.lens[s]), P.max_len);
  const int t0 = split * P.chunk, t1 = min(t0 + P.chunk, len);
  // columns of the workgroup's own sequence: heads 16 tile .. of its kv head
  const int own_heads = min(G - 16 * tile, 16), own_head = h * G + 16 * tile;
  const int slot = P.group > 1 ? split * (P.group + 1) : split;  // of its own record
  auto empty = [&](int from, int n) {  // records without tokens
    for (int e = tid; e < n * own_heads; e += kThr) {
      const int x = e / n, at = from + e - x * n;
      *reinterpret_cast<float2*>(P.part_ml + 2 * ((static_cast<int64_t>(s) * P.Hq + own_head + x) * P.slots + at)) =
          part_record(-INFINITY, 0.f);
    }
  };
  if (t0 >= t1) {  // uniform: nothing here
    if (P.slots == 1) {
      for (int e = tid; e < own_heads * (kD / 8); e += kThr)
        *reinterpret_cast<u32x4*>(P.out + s * P.o_ss + (own_head + e / (kD / 8)) * P.o_sh + 8 * (e % (kD / 8))) = u32x4{};
    } else {
      empty(slot, P.group > 1 ? P.group + 1 : 1);
    }
    return;
  }

  // ---- the split's pages; of the group's sequences where they end and how many pages they begin alike
  const int page0 = t0 >> st.lg, pages = ((t1 - 1) >> st.lg) - page0 + 1;
  const int* row = st.table + static_cast<int64_t>(s) * st.width + page0;
  for (int i = tid; i < min(pages, kMaxPages); i += kThr) sh.page[i] = page_id(st, row[i]);
  const int base = s - s % P.group, members = min(P.group, st.seqs - base);
  if (P.group > 1) {
    for (int j = wave; j < members; j += kWaves) {
      const int end = min(t0 + P.chunk, min(held(st, st.lens[base + j]), P.max_len));
      const int n = end > t0 ? min(((end - 1) >> st.lg) - page0 + 1, pages) : 0;
      const int* other = st.table + static_cast<int64_t>(base + j) * st.width + page0;
      int same = n;
      for (int i = 0; i < n; i += 64) {
        const int k = min(i + lane, n - 1);
        const uint64_t differs = wave_ballot(page_id(st, row[k]) != page_id(st, other[k]));
        if (differs) {
          same = min(n, i + static_cast<int>(__builtin_ctzll(differs)));
          break;
        }
      }
      if (lane == 0) {
        sh.end[j] = end;
        sh.same[j] = same;
      }
    }
  }
  __syncthreads();
  auto page_at = [&](int i) { return sh.page[i]; };
  auto all = [](int) { return 0; };
  int shared = t0, rank = 0, count = 0;  // shared tokens [t0, shared) of `count` sequences, this one the rank-th of them
  if (P.group > 1) {
    const int same = lane < members ? sh.same[lane] : 0;
    const uint32_t alike = static_cast<uint32_t>(wave_ballot(same > 0));
    int end = same > 0 ? min(sh.end[lane], (page0 + same) << st.lg) : 0x7fffffff;
#pragma unroll
    for (int x = 16; x; x >>= 1) end = min(end, __shfl_xor(end, x));
    end = __builtin_amdgcn_readfirstlane(end);
    if (__popc(alike) > 1 && end - t0 >= kStep) {  // (less is not worth a second part)
      shared = end;
      count = __popc(alike);
      rank = __popc(alike & ((1u << (s - base)) - 1));
      if (wave == 0 && same > 0) sh.member[__popc(alike & ((1u << lane) - 1))] = lane;
    }
    __syncthreads();
    empty(slot + 1 + count, P.group - count);
  }
  if (count) {
    const int cols = count * G;
    auto where = [&](int c, int& seq, int& head) {
      const int i = c * P.g_small >> 16;
      seq = base + sh.member[i];
      head = h * G + c - i * G;
    };
    const int part = ((shared - t0 + count - 1) / count + kChunk - 1) & ~(kChunk - 1);
    const int lo = min(t0 + rank * part, shared), hi = min(lo + part, shared);
    if (cols <= 16)
      attend<DT, 1, false>(P, sh, h, page0, lo, hi, hi, cols, slot + 1 + rank, where, all, page_at);
    else
      attend<DT, 2, false>(P, sh, h, page0, lo, hi, hi, cols, slot + 1 + rank, where, all, page_at);
  }
  auto own = [&](int c, int& seq, int& head) {
    seq = s;
    head = own_head + c;
  };
  if (shared >= t1)
    empty(slot, 1);
  else if (pages <= kMaxPages)
    attend<DT, 1, false>(P, sh, h, page0, shared, t1, t1, own_heads, slot, own, all, page_at);
  else  // (a plan without groups)
    attend<DT, 1, false>(P, sh, h, page0, shared, t1, t1, own_heads, slot, own, all,
                         [&](int i) { return page_id(st, row[i]); });
}

// The newest queries of every sequence, rows cu[s] .. of q: grid (splits, kv heads, sequences).
template <int DT>
__global__ __launch_bounds__(kThr, 2) void rows_kernel(DecodeArgs P) {
  __shared__ __align__(16) Staged sh;
  const Pages& st = P.st;
  const int tid = threadIdx.x;
  const int split = blockIdx.x, h = blockIdx.y, s = blockIdx.z, G = P.G;
  const int row0 = min(max(P.cu[s], 0), P.rows), m = min(max(P.cu[s + 1], row0), P.rows) - row0;
  const int len = held(st, st.lens[s]), qlen = min(m, len);
  if (P.fill) {  // rows of no sequence
    const int a = min(max(P.cu[0], 0), P.rows), e = min(max(P.cu[st.seqs], a), P.rows);
    const int64_t per = static_cast<int64_t>(P.Hq) * (kD / 8), n = (a + P.rows - e) * per;
    const int64_t block = blockIdx.x + static_cast<int64_t>(gridDim.x) * (blockIdx.y + gridDim.y * blockIdx.z);
    for (int64_t i = block * kThr + tid; i < n; i += static_cast<int64_t>(gridDim.x) * gridDim.y * gridDim.z * kThr) {
      const int64_t r = i / per, x = i - r * per, row = r < a ? r : r - a + e;
      *reinterpret_cast<u32x4*>(P.out + row * P.o_ss + x / (kD / 8) * P.o_sh + 8 * (x % (kD / 8))) = u32x4{};
    }
  }
  const int t0 = split * P.chunk, t1 = split == P.splits - 1 ? len : min(t0 + P.chunk, len);
  // queries that there are no tokens for, or none in this split
  const int from = t0 < t1 ? qlen : 0;
  for (int x = from * G + (tid >> 4); x < m * G; x += kThr / 16) {  // 16 lanes a row
    const int i = x / G;
    const int64_t row = row0 + i, head = h * G + x - i * G;
    if (P.slots == 1)
      *reinterpret_cast<u32x4*>(P.out + row * P.o_ss + head * P.o_sh + 8 * (tid & 15)) = u32x4{};
    else if ((tid & 15) == 0)
      *reinterpret_cast<float2*>(P.part_ml + 2 * ((row * P.Hq + head) * P.slots + split)) = part_record(-INFINITY, 0.f);
  }
  if (t0 >= t1 || !qlen) return;  // uniform

  const int page0 = t0 >> st.lg, pages = ((t1 - 1) >> st.lg) - page0 + 1;
  const int* table = st.table + static_cast<int64_t>(s) * st.width + page0;
  for (int i = tid; i < min(pages, kMaxPages); i += kThr) sh.page[i] = page_id(st, table[i]);
  __syncthreads();
  auto page_at = [&](int i) { return i < kMaxPages ? sh.page[i] : page_id(st, table[i]); };
#pragma unroll 1
  for (int col0 = 0; col0 < qlen * G; col0 += 32) {
    const int cols = min(qlen * G - col0, 32);
    auto where = [&](int c, int& row, int& head) {
      const int i = (col0 + c) / G;
      row = row0 + i;
      head = h * G + col0 + c - i * G;
    };
    auto sees = [&](int c) { return len - qlen + (col0 + c) / G + 1; };
    const int free = min(sees(0), t1);
    if (cols <= 16)
      attend<DT, 1, true>(P, sh, h, page0, t0, t1, free, cols, split, where, sees, page_at);
    else
      attend<DT, 2, true>(P, sh, h, page0, t0, t1, free, cols, split, where, sees, page_at);
  }
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
// splits, or many rows); otherwise they share one row, every eighth split each, and meet in LDS.
template <int DT, bool ONE>
__global__ __launch_bounds__(kThr) void join_kernel(JoinArgs A) {
  __shared__ __align__(16) float s_o[8][kD];
  __shared__ float s_l[8];
  const int tid = threadIdx.x, grp = tid >> 5, d = 4 * (tid & 31);
  const int row = ONE ? blockIdx.x * 8 + grp : blockIdx.x;
  if (row >= A.rows) return;  // (whole groups; with ONE no barrier follows)
  const int t = row / A.heads, head = row - t * A.heads;
  const float2* ml = reinterpret_cast<const float2*>(A.part_ml) + static_cast<int64_t>(row) * A.splits;
  const float2 first = (tid & 31) < A.splits ? ml[tid & 31] : part_record(-INFINITY, 0.f);
  if (A.cu && (t < A.cu[0] || t >= A.cu[A.n])) return;
  if (__shfl(first.y, 0, 32) < 0.f) return;  // the row is done (no sum of weights is negative)
  const float* po = A.part_o + static_cast<int64_t>(row) * A.splits * kD + d;
  float M = first.x;
  for (int i = (tid & 31) + 32; i < A.splits; i += 32) M = fmaxf(M, ml[i].x);
#pragma unroll
  for (int x = 16; x; x >>= 1) M = fmaxf(M, __shfl_xor(M, x));
  float L = 0.f;
  f32x4 o = f32x4{};
  for (int base = 0; base < A.splits; base += 32) {
    const int i = base + (tid & 31);
    const float2 r = base == 0 ? first : i < A.splits ? ml[i] : part_record(-INFINITY, 0.f);
    const float w = exp2_(r.x - M), wl = w * r.y;
    // the group's parts that are not empty (the rows of those were not written), four at a time on their way
    const uint64_t full = wave_ballot(r.x != -INFINITY && (ONE || (i & 7) == grp));
    for (uint32_t left = static_cast<uint32_t>(tid & 32 ? full >> 32 : full); left;) {
      f32x4 x[4];
      int at[4];
      bool is[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        is[k] = left != 0;
        at[k] = is[k] ? __builtin_ctz(left) : at[0];
        left &= left - 1;
        x[k] = *reinterpret_cast<const f32x4*>(po + static_cast<int64_t>(base + at[k]) * kD);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = __shfl(w, at[k], 32), fl = __shfl(wl, at[k], 32);
        L += is[k] ? fl : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = is[k] ? fmaf(f, x[k][j], o[j]) : o[j];
      }
    }
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
  int chunk, splits, group, slots;
};

size_t record_bytes(int64_t rows, int64_t slots) {
  return slots == 1 ? 0 : static_cast<size_t>(rows) * slots * (kD + 2) * 4;
}

// rows: of queries (x query heads), S of them where every sequence has one.
DecodePlan decode_plan(int64_t S, int64_t Hq, int64_t Hkv, int64_t max_len, int64_t rows, bool few = false) {
  const int64_t G = Hq / Hkv, tiles = few ? 1 : (G + 15) / 16, pairs = S * Hkv * tiles;
  const int64_t steps = (max_len + kStep - 1) / kStep;
  // Two workgroups a CU, the most that its registers hold at a time (32 x 8192 tokens, 32/8 heads: 186 us, with four 191,
  // 131072 tokens 100 and 108 us).  One split, which needs no join and shares nothing, where a workgroup a CU walks at most 8 steps
  // (32 x 1024: 24.2 us, in two splits 27.6), and up to 3 steps anyway.
  const int64_t cus = device_cu_count();
  int64_t splits = 1;
  if (steps > (pairs >= cus ? 8 : 3)) {
    splits = (2 * cus + pairs - 1) / pairs;
    splits = splits > steps ? steps : splits;
    splits = splits > kMaxSplits ? kMaxSplits : splits;
  }
  // page ids of a split fit their place whatever the page size: 16 tokens a page and the one that it begins in
  const int64_t most = (kMaxPages - 1) * 16 / kStep;
  DecodePlan p;
  auto cut = [&](int64_t chunk) {
    p.splits = static_cast<int>(steps <= chunk ? 1 : (steps + chunk - 1) / chunk);
    p.chunk = static_cast<int>(chunk * kStep);
  };
  const int64_t whole = (steps + splits - 1) / splits;
  cut(whole > most ? most : (whole < 1 ? 1 : whole));
  p.group = !few && p.splits > 1 && G <= 16 ? static_cast<int>(32 / G < S ? 32 / G : S) : 1;
  // Records for every sequence that might share pages, in every split, are bounded: smaller groups, then longer splits, whose
  // page ids past their place are read from the table (256 sequences of up to 131072 tokens, 32/8 heads: 345 MB with groups
  // of 8, 192 with 4; 2048 sequences alone 307 MB in 9 splits, 239 in 7).
  auto slots = [&]() { return static_cast<int64_t>(p.splits) * (p.group > 1 ? p.group + 1 : 1); };
  while (p.group > 1 && record_bytes(rows * Hq, slots()) > kMostBytes) p.group /= 2;
  if (p.group == 1 && record_bytes(rows * Hq, slots()) > kMostBytes) {
    const int64_t fit = static_cast<int64_t>(kMostBytes / (record_bytes(rows * Hq, 2) / 2));
    const int64_t fewer = fit > splits ? fit : splits;  // (no fewer than the workgroups need)
    cut((steps + fewer - 1) / fewer);
  }
  p.slots = static_cast<int>(slots());
  return p;
}

}  // namespace

int launch_join(const float* part_o, const float* part_ml, int64_t rows, int64_t splits, int64_t heads, void* out,
                int64_t o_st, int64_t o_sh, int dtype, const int* cu, int n, hipStream_t stream, const char* what) {
  const JoinArgs A{part_o, part_ml, static_cast<uint16_t*>(out), o_st, o_sh, cu, n, static_cast<int>(rows),
                   static_cast<int>(splits), static_cast<int>(heads)};
  // (16384 rows of 12 parts: 14 us more with a workgroup a row; 4096 of 32 8 us more with eight)
  const bool one = splits <= 8 || rows >= 256 * splits;
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

size_t few_rows_bytes(int64_t rows, int64_t S, int64_t Hq, int64_t Hkv, int64_t max_len) {
  return record_bytes(rows * Hq, decode_plan(S, Hq, Hkv, max_len, rows, true).slots);
}

int launch_few_rows(const lkv_pages* p, int64_t layer, const void* q, const int64_t* q_strides, int64_t rows, int64_t Hq,
                    const int32_t* cu, int64_t max_len, float scale, void* out, const int64_t* out_strides, int fill,
                    void* workspace, size_t workspace_bytes, hipStream_t s, const char* what) {
  const size_t need = few_rows_bytes(rows, p->seqs, Hq, p->kv_heads, max_len);
  LKV_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
              "%s: a 16-byte aligned workspace of %zu bytes required, got %zu", what, need, workspace_bytes);
  const DecodePlan plan = decode_plan(p->seqs, Hq, p->kv_heads, max_len, rows, true);
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
  A.G = static_cast<int>(Hq / p->kv_heads);
  A.max_len = static_cast<int>(max_len);
  A.chunk = plan.chunk;
  A.splits = A.slots = plan.splits;
  A.cu = cu;
  A.rows = static_cast<int>(rows);
  A.fill = fill;
  A.scale_log2 = scale * kLog2e;
  A.part_o = static_cast<float*>(workspace);
  A.part_ml = A.part_o + static_cast<size_t>(rows * Hq) * plan.slots * kD;
  const dim3 grid(static_cast<unsigned>(plan.splits), static_cast<unsigned>(p->kv_heads), static_cast<unsigned>(p->seqs));
  if (p->dtype == LKV_DTYPE_F16)
    hipLaunchKernelGGL(rows_kernel<LKV_DTYPE_F16>, grid, dim3(kThr), 0, s, A);
  else
    hipLaunchKernelGGL(rows_kernel<LKV_DTYPE_BF16>, grid, dim3(kThr), 0, s, A);
  LKV_LAUNCH_CHECK(what);
  if (plan.slots == 1) return LKV_OK;
  return launch_join(A.part_o, A.part_ml, rows * Hq, plan.slots, Hq, out, A.o_ss, A.o_sh, p->dtype, cu,
                     static_cast<int>(p->seqs), s, what);
}

}  // namespace pages
}  // namespace lkv

using namespace lkv;
using namespace lkv::pages;

extern "C" size_t lkv_pages_decode_attn_workspace_bytes(int64_t seqs, int64_t Hq, int64_t Hkv, int64_t max_len) {
  if (seqs < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || max_len < 0) return 0;
  return record_bytes(seqs * Hq, decode_plan(seqs, Hq, Hkv, max_len, seqs).slots);
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
  const DecodePlan plan = decode_plan(p->seqs, Hq, p->kv_heads, max_len, p->seqs);
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
  A.group = plan.group;
  A.g_small = static_cast<int>(65536 / G + 1);
  A.slots = plan.slots;
  A.max_len = static_cast<int>(max_len);
  A.chunk = plan.chunk;
  A.splits = plan.splits;
  A.scale_log2 = scale * kLog2e;
  A.part_o = static_cast<float*>(workspace);
  A.part_ml = A.part_o + static_cast<size_t>(p->seqs * Hq) * plan.slots * kD;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(plan.splits), static_cast<unsigned>(p->kv_heads * tiles),
                  static_cast<unsigned>(p->seqs));
  if (p->dtype == LKV_DTYPE_F16)
    hipLaunchKernelGGL(split_kernel<LKV_DTYPE_F16>, grid, dim3(kThr), 0, s, A);
  else
    hipLaunchKernelGGL(split_kernel<LKV_DTYPE_BF16>, grid, dim3(kThr), 0, s, A);
  LKV_LAUNCH_CHECK(what);
  if (plan.slots == 1) return LKV_OK;
  return launch_join(A.part_o, A.part_ml, p->seqs * Hq, plan.slots, Hq, out, A.o_ss, A.o_sh, p->dtype, nullptr, 0, s,
                     "pages_decode_attn join");
}
