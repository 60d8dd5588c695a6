// Causal attention of many query rows in 16 bits: packed prompts (lkv_packed_attn), and packed chunks over the paged KV cache
// (lkv_pages_prefill_attn).
//
// A workgroup of 8 waves owns 256 columns of a kv head of one sequence, column c the query row (query c / G, head c % G), so
// that its columns end at nearly the same token; a wave has 32.  It walks the tiles of 64 tokens that its columns see.  Each
// tile's rows of keys and values are copied to LDS once for all 8 waves, through buffer descriptors that end with the
// sequence (rows past it read as zeros).  Every wave then runs, on v_mfma_f32_32x32x16,
//   scores^T (32 tokens x 32 columns): A = keys from LDS, B = the wave's queries (registers),
//   softmax: a lane holds 32 of the 64 scores of one column (lane ^ 32 the others),
//   out^T (32 dims x 32 columns) += A = values from LDS, transposed as they are read (ds_read_b64_tr_b16), B = the weights
//   from the lane's own registers (the values' token order is the order in which a lane holds its scores).
// A wave's 32 products a tile are in two stretches of 16 with vector work between them: scores of the next tile beside the
// exponentials of this one, values of this one beside the next one's offsets and the staging.  The running offset moves
// only when a weight passes 2^15, so that most tiles need no max over lanes and no rescale.
//
// A masked token has weight 0, but 0 times an infinite or NaN value is not 0.  Where a row ends up with such a number its
// workgroup goes through the piece again with care: values that are no numbers count as 0 in the masked tiles' products, and
// a second product counts, of each kind, those that a column sees.
#include "pages_common.h"

namespace lkv {
namespace pages {
namespace {

constexpr int kWaves = 8;
constexpr int kThr = 64 * kWaves;
constexpr int kCols = 32 * kWaves;
constexpr int kTile = 64;         // tokens of a tile
constexpr int kKRow = kD + 8;     // 16-bit numbers of a staged key row: 16 rows' 16-byte reads fall in distinct banks
constexpr int kVRow = kD + 32;    // and of a value row: the transposing read's 4 rows of 64 bytes do
constexpr int kKBuf = kTile * kKRow, kVBuf = kTile * kVRow;
constexpr int kXcds = 8;
constexpr int kManyChunk = 8;     // fewest tiles of a split
constexpr int kAgain = 128;       // words of marks (rounds past 4096 share them: gone through again without need)

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

__device__ __forceinline__ float half_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

struct Args {
  const uint16_t* k;   // packed rows
  const uint16_t* v;
  int64_t k_sh, v_sh;  // strides of head and row
  int k_st, v_st;
  const uint16_t* q;
  int64_t q_st, q_sh;
  uint16_t* out;
  int64_t o_st, o_sh;
  const int* cu;
  int B, rows;         // sequences, packed rows
  Pages st;            // PAGED: the store, and the layer's pages
  const uint16_t* kv;
  int H, G, Hq;
  int chunk, splits;   // tiles of a split
  int fill;
  float scale_log2;
  float* part_o;       // [rows * Hq][splits][128]
  float* part_ml;      // [rows * Hq][splits][2]
};

// The kernel's arguments, read where they stand: what a piece needs once is not held in registers through its tiles.
typedef const __attribute__((address_space(4))) Args* ArgsPtr;
__device__ __forceinline__ ArgsPtr args_again() {
  ArgsPtr p = (ArgsPtr)__builtin_amdgcn_kernarg_segment_ptr();
  __asm__ volatile("" : "+s"(p));
  return p;
}

// Column tiles of sequence b with more than x tokens to read, of tiles with m rows in all and q of them queries of the last
// of len tokens.
__device__ __forceinline__ int tiles_over(int x, int len, int m, int G) {
  const int q = min(m, len), all = (m * G + kCols - 1) / kCols;
  const int y = x - (len - q);
  const int under = y <= 0 ? 0 : y >= q ? all : min(all, y * G / kCols);
  return x < 0 ? all : all - under;
}
__device__ __forceinline__ int wave_total(int v) {
#pragma unroll
  for (int x = 32; x; x >>= 1) v += __shfl_xor(v, x);
  return __builtin_amdgcn_readfirstlane(v);
}

// Goes through the workgroup's pieces.  CARE: those that the first time marked in s_again, with care for values that are no
// numbers.  Returns whether any is to be gone through again.
template <int DT, bool PAGED, bool CARE>
__device__ __forceinline__ bool go_through(const Args& P, uint16_t* smem, const int* s_len, const int* s_rows,
                                           uint32_t* s_again, int wave, int longest, int pieces) {
  uint16_t* const sK = smem;
  uint16_t* const sV = smem + 2 * kKBuf;
  const int lane = lane_prefix(~0ull);
  const int c32 = lane & 31, hf = lane >> 5;
  const int G = P.G;
  bool again = false;

  // ---- staging: thread's rows 8 wave + lane / 16 and 4 further, piece lane % 16 of 16 bytes
  const int srow = lane >> 4, spiece = 8 * (lane & 15);
  const int64_t run = PAGED ? run_numbers(P.st) : 0;
  const int k_st = PAGED ? kD : P.k_st, v_st = PAGED ? kD : P.v_st;
  const int koff = 2 * (srow * k_st + spiece), voff = PAGED ? koff : 2 * (srow * v_st + spiece);
  uint16_t* const kdst = sK + (8 * wave + srow) * kKRow + spiece;
  uint16_t* const vdst = sV + (8 * wave + srow) * kVRow + spiece;
  const uint16_t* const krow = sK + c32 * kKRow + 8 * hf;
  // a transposing read: lane's 8 bytes of token 4 hf + (lane % 16) / 4, dims 16 ((lane / 16) % 2) + 4 (lane % 4)
  const uint16_t* const vrow = sV + (4 * hf + ((lane & 15) >> 2)) * kVRow + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);

  // The workgroups stay and take their pieces of work in turn, the longest first and the order reversed in every second
  // round, so that each gets as much.  Workgroups go to the XCDs round-robin, and the column tiles of one (sequence, kv
  // head) read the same rows: where the numbers allow it a head is taken on one XCD.
  const int lanes = gridDim.x % kXcds == 0 && P.H % kXcds == 0 ? kXcds : 1;
  const int heads_lane = P.H / lanes;
  const int width = static_cast<int>(gridDim.x) / lanes;
  const int own = static_cast<int>(blockIdx.x) / lanes, xcd = static_cast<int>(blockIdx.x) % lanes;
  const int per_lane = pieces * P.splits * heads_lane;
#pragma unroll 1
  for (int round = 0; round * width < per_lane; ++round) {
    const int pos = round * width + ((round & 1) ? width - 1 - own : own);
    if (pos >= per_lane) continue;  // uniform
    if (CARE && !((s_again[(round >> 5) & (kAgain - 1)] >> (round & 31)) & 1)) continue;  // uniform
    const int ps = __builtin_amdgcn_readfirstlane(pos / heads_lane);
    const int h = (pos - ps * heads_lane) * lanes + xcd;
    const int piece = __builtin_amdgcn_readfirstlane(ps / P.splits), split = ps - piece * P.splits;
    // ---- the piece-th column tile by falling length: its length in tiles of tokens, then its place among those
    int b = 0, tile;
    {
      int lo = -1, hi = (longest + kTile - 1) / kTile, over = 0;  // more than `piece` tiles over 64 lo, none over 64 hi
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        int n = 0;
        for (int i = lane; i < P.B; i += 64) n += tiles_over(mid * kTile, s_len[i], s_rows[i], G);
        n = wave_total(n);
        if (n > piece) {
          lo = mid;
        } else {
          hi = mid;
          over = n;
        }
      }
      const int x = lo < 0 ? -1 : lo * kTile, x2 = hi * kTile;
      int rank = piece - over;
      tile = 0;
      for (int base = 0; base < P.B; base += 64) {
        const int i = base + lane;
        const int high = i < P.B ? tiles_over(x2, s_len[i], s_rows[i], G) : 0;
        const int n = i < P.B ? tiles_over(x, s_len[i], s_rows[i], G) - high : 0;
        int sum = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const int y = __shfl_up(sum, d);
          if (lane >= d) sum += y;
        }
        const uint64_t past = wave_ballot(sum > rank);
        if (past) {
          const int at = __builtin_ctzll(past);
          b = base + at;
          const int before = __builtin_amdgcn_readlane(sum - n, at);
          // its tiles from the longest: `high` are longer than these
          const int all = (s_rows[b] * G + kCols - 1) / kCols;
          tile = all - 1 - __builtin_amdgcn_readlane(high, at) - (rank - before);
          break;
        }
        rank -= __builtin_amdgcn_readlane(sum, 63);
      }
      b = __builtin_amdgcn_readfirstlane(b);
      tile = __builtin_amdgcn_readfirstlane(tile);
    }
    const int len = __builtin_amdgcn_readfirstlane(s_len[b]), m_rows = __builtin_amdgcn_readfirstlane(s_rows[b]);
    const int row0 = __builtin_amdgcn_readfirstlane(min(max(P.cu[b], 0), P.rows));
    const int qlen = min(m_rows, len), cols = m_rows * G;
    const int col0 = tile * kCols;
    const int q_first = __builtin_amdgcn_readfirstlane(col0 / G);
    const int last = min(__builtin_amdgcn_readfirstlane((col0 + kCols - 1) / G), qlen - 1);  // its last query
    const int kend = last >= q_first ? len - qlen + last + 1 : 0;
    // tiles [blk0, blk0 + nt) of 64 tokens: what the piece's last column sees, of the split's
    const int blk0 = split * P.chunk;
    const int all_t = (kend + kTile - 1) / kTile;
    const int nt = max((split == P.splits - 1 ? all_t : min(blk0 + P.chunk, all_t)) - blk0, 0);

    // ---- a tile's rows: descriptors of the wave's 8 rows of keys and values
    u32x4 kw[2], vw[2];
    auto first_of = [&](int t) { return (blk0 + t) * kTile + 8 * wave; };
    auto page_of = [&](int t) {  // (past the last tile: the last page, of which nothing is read)
      const int e = min(first_of(t), len - 1) >> P.st.lg;
      return page_id(P.st, P.st.table[static_cast<int64_t>(b) * P.st.width + e]);
    };
    auto rows_of = [&](int t) { return t < nt ? min(max(len - first_of(t), 0), 8) : 0; };
    auto load_rows = [&](u32x4 (&w)[2], const uint16_t* p, int n, int stride, int off) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int rows = min(max(n - 4 * j, 0), 4);
        const int bytes = rows ? 2 * ((rows - 1) * stride + kD) : 0;
        const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p + (rows ? 4 * j * stride : 0)), 0, bytes,
                                                         0x00020000);
        w[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
      }
    };
    auto load_k = [&](int t, int page) {
      const int n = rows_of(t), at = first_of(t);
      load_rows(kw, PAGED ? P.kv + (static_cast<int64_t>(page) * 2 * P.H + h) * run + (at & (page_size(P.st) - 1)) * kD
                          : P.k + (n ? static_cast<int64_t>(row0 + at) * k_st : 0) + h * P.k_sh, n, k_st, koff);
    };
    auto load_v = [&](int t, int page) {
      const int n = rows_of(t), at = first_of(t);
      load_rows(vw, PAGED ? P.kv + ((static_cast<int64_t>(page) * 2 + 1) * P.H + h) * run + (at & (page_size(P.st) - 1)) * kD
                          : P.v + (n ? static_cast<int64_t>(row0 + at) * v_st : 0) + h * P.v_sh, n, v_st, voff);
    };
    auto stage_k = [&](int t, int j) {
      *reinterpret_cast<u32x4*>(kdst + (t & 1) * kKBuf + 4 * j * kKRow) = kw[j];
    };
    auto stage_v = [&](int t, int j) {
      *reinterpret_cast<u32x4*>(vdst + (t & 1) * kVBuf + 4 * j * kVRow) = vw[j];
    };
    u32x4 k1[2];
    int page1 = 0, page2 = 0;  // pages of the wave's rows in the next tiles
    auto first_loads = [&]() {
      if (!nt) return;
      int page0 = 0;
      if constexpr (PAGED) {
        page0 = page_of(0);
        page1 = page_of(1);
        page2 = page_of(2);
      }
      load_k(1, page1);
      k1[0] = kw[0];
      k1[1] = kw[1];
      load_k(0, page0);
      load_v(0, page0);
    };
    if constexpr (!CARE) first_loads();
    // ---- the lane's column: query qs, head qh
    const int col = col0 + 32 * wave + c32, qs = col / G, qh = col - qs * G;
    const bool ok = col < cols && qs < qlen;
    const int lim = ok ? len - qlen + qs + 1 : 0x7fffffff;  // tokens it sees
    u32x4 qf[8];  // B: dims 16 kb + 8 hf ..
    {
      const ArgsPtr Z = args_again();
      const uint16_t* p = Z->q + (row0 + qs) * Z->q_st + (static_cast<int64_t>(h) * G + qh) * Z->q_sh + 8 * hf;
#pragma unroll
      for (int kb = 0; kb < 8; ++kb) qf[kb] = ok ? *reinterpret_cast<const u32x4*>(p + 16 * kb) : u32x4{};
    }
    // tokens that every column of the wave sees
    const int wq = __builtin_amdgcn_readfirstlane((col0 + 32 * wave) / G);
    const int lim_min = wq < qlen ? len - qlen + wq + 1 : 0x7fffffff;

    float m, l;
    f32x16 o[4];   // dims 32 db + 8 (i / 4) + 4 hf + i % 4
    f32x16 sc[2];  // scores of tokens 32 kt + 8 (i / 4) + 4 hf + i % 4
    float s[32];   // log2 weights of the present tile, relative to m
    float ws[2];
    u32x4 pf[4];   // its weights
    constexpr int kAhead = 4;  // operands on their way from LDS
    u32x4 fr[kAhead];
    // operand i of the 16 score products (tile t's keys) and of the 16 value products
    auto key_op = [&](int i, int t) {
      return *reinterpret_cast<const u32x4*>(krow + (t & 1) * kKBuf + 32 * (i & 1) * kKRow + 16 * (i >> 1));
    };
    auto value_op = [&](int i, int t) {
      const uint16_t* p = vrow + (t & 1) * kVBuf + 16 * (i >> 2) * kVRow + 32 * (i & 3);
      const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p)));
      const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * kVRow)));
      return u32x4{lo.x, lo.y, hi.x, hi.y};
    };
    const float kc = P.scale_log2;
    auto score_products = [&](int t) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i & 1] = mfma32<DT>(key_op(i, t), qf[i >> 1], i < 2 ? f32x16{} : sc[i & 1]);
    };
    // masks and a new offset, where a column of the wave needs one
    auto general = [&](int t) {
      const int left = lim - (blk0 + t) * kTile - 4 * hf;
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float x = sc[e >> 4][e & 15] * kc;
        s[e] = 8 * (e >> 2) + (e & 3) < left ? x : -INFINITY;
        mx = fmaxf(mx, s[e]);
      }
      mx = half_max(mx);
      const float mn = mx - m > kMaxWeight ? mx - kTopWeight : m;
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float alpha = exp2_(m - mu);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < 4; ++db) o[db] = o[db] * alpha;
#pragma unroll
      for (int e = 0; e < 32; ++e) s[e] -= mu;
    };
    // weights 2 i, 2 i + 1 of the present tile, into the value operand
    auto weights = [&](int i) {
      const float a = exp2_(s[2 * i]), c = exp2_(s[2 * i + 1]);
      ws[0] += a;
      ws[1] += c;
      uint32_t u = pack<DT>(a, c);
      __asm__ volatile("" : "+v"(u));  // (no instruction: keeps the work beside the product that it stands next to)
      pf[i >> 2][i & 3] = u;
    };
    m = ok ? -INFINITY : 0.f;  // a column that is no row keeps offset 0 over zero scores
    l = 0.f;
#pragma unroll
    for (int db = 0; db < 4; ++db) o[db] = f32x16{};
    if constexpr (CARE) {
#pragma unroll 1
      for (int t = 0; t < nt; ++t) {
        int page0 = 0;
        if constexpr (PAGED) page0 = page_of(t);
        load_k(t, page0);
        load_v(t, page0);
        __syncthreads();  // the buffers are free
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          stage_k(0, j);
          stage_v(0, j);
        }
        __syncthreads();
        score_products(0);
        general(t);
        ws[0] = ws[1] = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) weights(i);
        l += ws[0] + ws[1];
        __builtin_amdgcn_sched_barrier(0);
        constexpr uint32_t kInf = DT == LKV_DTYPE_F16 ? 0x7c00u : 0x7f80u;
        constexpr uint32_t kOne = DT == LKV_DTYPE_F16 ? 0x3c00u : 0x3f80u;  // 1
        constexpr uint32_t k128 = DT == LKV_DTYPE_F16 ? 0x5800u : 0x4300u;  // 128
        constexpr uint32_t k129 = DT == LKV_DTYPE_F16 ? 0x5808u : 0x4301u;  // 129
#pragma unroll
        for (int db = 0; db < 4; ++db) {
          f32x16 count = f32x16{};  // +inf counts 1, -inf 128, NaN both
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const u32x4 raw = value_op(4 * ks + db, 0);
            u32x4 fine, kind, seen;
            int left = lim - (blk0 + t) * kTile - 4 * hf;
            __asm__ volatile("" : "+v"(left));  // (its comparisons are made where they are used)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t f = 0, n = 0, z = 0;
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const uint32_t y = (raw[j] >> (16 * x)) & 0xffffu, a = y & 0x7fffu;
                f |= (a >= kInf ? 0u : y) << (16 * x);
                n |= (a < kInf ? 0u : a > kInf ? k129 : (y >> 15) ? k128 : kOne) << (16 * x);
                const int e = 2 * j + x;  // token 16 ks + 4 hf + e % 4 + 8 (e / 4)
                z |= (16 * ks + (e & 3) + 8 * (e >> 2) < left ? kOne : 0u) << (16 * x);
              }
              fine[j] = f;
              kind[j] = n;
              seen[j] = z;
            }
            o[db] = mfma32<DT>(fine, pf[ks], o[db]);
            count = mfma32<DT>(kind, seen, count);
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float minus = floorf(count[i] * (1.f / 128.f)), plus = count[i] - 128.f * minus;
            if (plus > 0.f) o[db][i] += INFINITY;
            if (minus > 0.f) o[db][i] -= INFINITY;
          }
        }
      }
    } else {
      // ---- tile 0 (and the keys of tile 1)
      __syncthreads();  // the buffers are free
      if (nt) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          stage_k(0, j);
          stage_v(0, j);
        }
        kw[0] = k1[0];
        kw[1] = k1[1];
#pragma unroll
        for (int j = 0; j < 2; ++j) stage_k(1, j);
        load_v(1, page1);
        load_k(2, page2);
        if constexpr (PAGED) {
          page1 = page2;
          page2 = page_of(3);
        }
      }
      __syncthreads();
      if (nt) {
        score_products(0);
        general(0);
      }
      __syncthreads();  // (the keys of tile 0 are overwritten next)
      // ---- A tile is two stretches of 16 products, each with vector work between them: the scores of tile t + 1 beside
      // the weights of tile t, then the values of tile t beside the offsets of tile t + 1 and the staging of the next
      // tiles.  Keys and values have two buffers: what a tile overwrites was last read in the tile before.  (Past the last
      // tile the scores are of zeros, unused.)
#pragma unroll 1
      for (int t = 0; t < nt; ++t) {
        ws[0] = ws[1] = 0.f;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) fr[i] = key_op(i, t + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          sc[i & 1] = mfma32<DT>(fr[i % kAhead], qf[i >> 1], i < 2 ? f32x16{} : sc[i & 1]);
          fr[i % kAhead] = i + kAhead < 16 ? key_op(i + kAhead, t + 1) : value_op(i + kAhead - 16, t);
          weights(i);
          __builtin_amdgcn_sched_barrier(0);
        }
        l += ws[0] + ws[1];
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          o[i & 3] = mfma32<DT>(fr[i % kAhead], pf[i >> 2], o[i & 3]);
          if (i + kAhead < 16) fr[i % kAhead] = value_op(i + kAhead, t);
          if ((i & 3) == 0) {
            if (i < 8)
              stage_k(t + 2, i >> 2);
            else
              stage_v(t + 1, (i >> 2) - 2);
          }
          s[2 * i] = fmaf(sc[i >> 3][2 * i & 15], kc, -m);
          s[2 * i + 1] = fmaf(sc[i >> 3][(2 * i + 1) & 15], kc, -m);
          mx = fmaxf(fmaxf(mx, s[2 * i]), s[2 * i + 1]);
        }
        load_v(t + 2, page1);
        load_k(t + 3, page2);
        if constexpr (PAGED) {
          page1 = page2;
          page2 = page_of(t + 4);
        }
        if (t + 1 < nt && ((blk0 + t + 2) * kTile > lim_min || wave_ballot(mx > kMaxWeight) != 0)) general(t + 1);  // uniform
        __syncthreads();
      }
      float odd = 0.f;
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) odd = fmaf(o[db][i], 0.f, odd);  // (an infinity or NaN times 0 is NaN, and NaN != 0)
      if (__syncthreads_or(ok && odd != 0.f)) {
        if (wave == 0 && lane == 0) s_again[(round >> 5) & (kAgain - 1)] |= 1u << (round & 31);
        again = true;
      }
    }

    const ArgsPtr Z = args_again();
    // (what follows from the lane is computed again here, from a copy: it needs no registers before)
    int out_lane = lane_prefix(~0ull);
    __asm__ volatile("" : "+v"(out_lane));
    const int ox = out_lane & 31, oh = out_lane >> 5;
    const int out_col = col0 + 32 * wave + ox;
    const int out_q = out_col / G, out_h = out_col - out_q * G;
    const int64_t out_row = row0 + out_q, out_head = static_cast<int64_t>(h) * G + out_h;
    // ---- out: a wave's 32 rows through its part of LDS (the tiles are done with), so that a row goes out whole
    l = half_sum(l);
    __syncthreads();
    constexpr int kOutRow = 272;  // bytes of a staged row: 256 and a shift of the banks
    static_assert(32 * kOutRow * kWaves <= 2 * (2 * kKBuf + 2 * kVBuf), "every wave's rows fit");
    char* const rows = reinterpret_cast<char*>(smem) + 32 * kOutRow * wave;
    char* const mine_row = rows + kOutRow * ox;
    // the 16 bytes that a lane takes of row 4 j + lane / 16 (a row's address and whether it exists come from its lane)
    auto out_rows = [&](int64_t at, bool exists, auto put) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = 4 * j + (out_lane >> 4);
        const u32x4 v = *reinterpret_cast<const u32x4*>(rows + kOutRow * row + 16 * (out_lane & 15));
        const int64_t to = __shfl(static_cast<long long>(at), row);
        if (__shfl(static_cast<int>(exists), row)) put(to, v);
      }
    };
    if (Z->splits == 1) {
      const bool some = ok && l != 0.f;
      const float inv = some ? 1.f / l : 0.f;
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = some ? o[db][4 * k + i] * inv : 0.f;
          *reinterpret_cast<uint2*>(mine_row + 2 * (32 * db + 8 * k + 4 * oh)) =
              uint2{pack<DT>(x[0], x[1]), pack<DT>(x[2], x[3])};
        }
      out_rows(out_row * Z->o_st + out_head * Z->o_sh, out_col < cols, [&](int64_t to, const u32x4& v) {
        *reinterpret_cast<u32x4*>(Z->out + to + 8 * (out_lane & 15)) = v;
      });
    } else {
      const int64_t at = (out_row * Z->Hq + out_head) * Z->splits + split;
      const bool some = ok && nt > 0;
      if (oh == 0 && out_col < cols)
        *reinterpret_cast<float2*>(Z->part_ml + 2 * at) = some ? part_record(m, l) : part_record(-INFINITY, 0.f);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const f32x16& x = o[2 * half + db];
            *reinterpret_cast<f32x4*>(mine_row + 4 * (32 * db + 8 * k + 4 * oh)) =
                f32x4{x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]};
          }
        out_rows(at * kD + 64 * half, some, [&](int64_t to, const u32x4& v) {
          *reinterpret_cast<u32x4*>(Z->part_o + to + 4 * (out_lane & 15)) = v;
        });
      }
    }
  }
  return again;
}

template <int DT, bool PAGED>
__global__ __launch_bounds__(kThr, 1) void prefill_kernel(Args P) {
  __shared__ __align__(16) uint16_t smem[2 * kKBuf + 2 * kVBuf];
  __shared__ int s_len[kMaxSeqs], s_rows[kMaxSeqs];
  __shared__ uint32_t s_again[kAgain];  // pieces to go through again, by round
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tid = threadIdx.x, lane = tid & 63;
  const int G = P.G;

  // ---- every sequence's tokens and rows; the longest
  int longest = 0;
  for (int b = tid; b < P.B; b += kThr) {
    const int a = min(max(P.cu[b], 0), P.rows), e = min(max(P.cu[b + 1], a), P.rows);
    s_rows[b] = e - a;
    s_len[b] = PAGED ? held(P.st, P.st.lens[b]) : e - a;
  }
  if (tid < kAgain) s_again[tid] = 0;
  __syncthreads();
  int pieces = 0;  // column tiles of all sequences
  for (int b = lane; b < P.B; b += 64) {
    longest = max(longest, s_len[b]);
    pieces += tiles_over(-1, s_len[b], s_rows[b], G);
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) longest = max(longest, __shfl_xor(longest, x));
  longest = __builtin_amdgcn_readfirstlane(longest);
  pieces = wave_total(pieces);

  if (go_through<DT, PAGED, false>(P, smem, s_len, s_rows, s_again, wave, longest, pieces)) {
    __syncthreads();
    go_through<DT, PAGED, true>(P, smem, s_len, s_rows, s_again, wave, longest, pieces);
  }

  // ---- rows of no sequence
  const ArgsPtr Z = args_again();
  if (Z->fill) {
    const int a = min(max(Z->cu[0], 0), Z->rows), e = min(max(Z->cu[Z->B], a), Z->rows);
    const int64_t per = static_cast<int64_t>(Z->Hq) * (kD / 8), n = (a + Z->rows - e) * per;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThr + tid; i < n; i += static_cast<int64_t>(gridDim.x) * kThr) {
      const int64_t r = i / per, x = i - r * per;
      const int64_t row = r < a ? r : r - a + e;
      *reinterpret_cast<u32x4*>(Z->out + row * Z->o_st + x / (kD / 8) * Z->o_sh + 8 * (x % (kD / 8))) = u32x4{};
    }
  }
}

struct Plan {
  int64_t pieces;  // most column tiles of a kv head, over all sequences
  int chunk, splits;
};

Plan make_plan(int64_t rows, int64_t B, int64_t Hq, int64_t Hkv, int64_t max_new, int64_t max_len) {
  const int64_t G = Hq / Hkv;
  const int64_t each = B * ((max_new * G + kCols - 1) / kCols), packed = rows * G / kCols + B;
  Plan p;
  p.pieces = each < packed ? each : packed;
  p.pieces = p.pieces < 1 ? 1 : p.pieces;
  const int64_t cus = device_cu_count(), tiles = (max_len + kTile - 1) / kTile;
  int64_t splits = cus / (p.pieces * Hkv);
  const int64_t most = tiles / kManyChunk;
  splits = splits > most ? most : splits;
  splits = splits < 1 ? 1 : splits;
  const int64_t chunk = (tiles + splits - 1) / splits;
  p.chunk = static_cast<int>(chunk < 1 ? 1 : chunk);
  p.splits = static_cast<int>(tiles <= p.chunk ? 1 : (tiles + p.chunk - 1) / p.chunk);
  return p;
}

size_t plan_bytes(const Plan& p, int64_t rows, int64_t Hq) {
  return p.splits == 1 ? 0 : static_cast<size_t>(rows * Hq) * p.splits * (kD + 2) * 4;
}

template <bool PAGED>
int launch(Args A, const Plan& p, int dtype, void* workspace, size_t workspace_bytes, hipStream_t s, const char* what) {
  const size_t need = plan_bytes(p, A.rows, A.Hq);
  LKV_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
              "%s: a 16-byte aligned workspace of %zu bytes required, got %zu", what, need, workspace_bytes);
  A.chunk = p.chunk;
  A.splits = p.splits;
  A.part_o = static_cast<float*>(workspace);
  A.part_ml = A.part_o + static_cast<size_t>(A.rows) * A.Hq * p.splits * kD;
  const int64_t work = p.pieces * p.splits * A.H, cus = device_cu_count();
  const int64_t most = (static_cast<int64_t>(A.rows) * A.G / kCols + A.B) * p.splits * A.H;  // whatever cu holds
  LKV_REQUIRE(most < (1ll << 30), "%s: %lld pieces of work", what, (long long)most);
  const dim3 grid(static_cast<unsigned>(work < cus ? work : cus));
  if (dtype == LKV_DTYPE_F16)
    hipLaunchKernelGGL((prefill_kernel<LKV_DTYPE_F16, PAGED>), grid, dim3(kThr), 0, s, A);
  else
    hipLaunchKernelGGL((prefill_kernel<LKV_DTYPE_BF16, PAGED>), grid, dim3(kThr), 0, s, A);
  LKV_LAUNCH_CHECK(what);
  if (p.splits == 1) return LKV_OK;
  return launch_join(A.part_o, A.part_ml, static_cast<int64_t>(A.rows) * A.Hq, p.splits, A.Hq, A.out, A.o_st, A.o_sh,
                     dtype, A.cu, A.B, s, what);
}

int check_queries(int64_t rows, int64_t Hq, int64_t Hkv, const int32_t* cu, const char* what) {
  LKV_REQUIRE(Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Hq < (1 << 20), "%s: %lld query heads over %lld kv heads", what,
              (long long)Hq, (long long)Hkv);
  LKV_REQUIRE(rows >= 0 && rows < (1ll << 30) && rows * Hq < (1ll << 30), "%s: %lld rows of %lld heads", what,
              (long long)rows, (long long)Hq);
  LKV_REQUIRE(cu && aligned4(cu), "%s: cu must be 4-byte aligned", what);
  return LKV_OK;
}

}  // namespace
}  // namespace pages
}  // namespace lkv

using namespace lkv;
using namespace lkv::pages;

extern "C" size_t lkv_packed_attn_workspace_bytes(int64_t rows, int64_t B, int64_t Hq, int64_t Hkv, int64_t max_len) {
  if (rows < 1 || B < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || max_len < 0) return 0;
  const int64_t most = max_len < rows ? max_len : rows;
  return plan_bytes(make_plan(rows, B, Hq, Hkv, most, most), rows, Hq);
}

extern "C" int lkv_packed_attn(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                               const void* v, const int64_t* v_strides, int dtype, int64_t rows, int64_t Hq, int64_t Hkv,
                               const int32_t* cu, int64_t B, int64_t max_len, float scale, void* out,
                               const int64_t* out_strides, int fill, void* workspace, size_t workspace_bytes,
                               void* stream) {
  const char* what = "packed_attn";
  LKV_REQUIRE(dtype == LKV_DTYPE_F16 || dtype == LKV_DTYPE_BF16, "%s: dtype %d (float16 or bfloat16)", what, dtype);
  if (int rc = check_queries(rows, Hq, Hkv, cu, what)) return rc;
  LKV_REQUIRE(B >= 1 && B <= kMaxSeqs, "%s: B=%lld must be 1 .. %d", what, (long long)B, kMaxSeqs);
  LKV_REQUIRE(max_len >= 0, "%s: max_len=%lld", what, (long long)max_len);
  if (rows == 0) return LKV_OK;
  if (int rc = check_rows(q, q_strides, what, "q")) return rc;
  if (int rc = check_rows(k, k_strides, what, "k")) return rc;
  if (int rc = check_rows(v, v_strides, what, "v")) return rc;
  if (int rc = check_rows(out, out_strides, what, "out")) return rc;
  LKV_REQUIRE(k_strides[0] < (1ll << 26) && v_strides[0] < (1ll << 26), "%s: strides of rows of k or v past 2^26", what);
  Args A{};
  A.q = static_cast<const uint16_t*>(q);
  A.q_st = q_strides[0];
  A.q_sh = q_strides[1];
  A.k = static_cast<const uint16_t*>(k);
  A.k_st = static_cast<int>(k_strides[0]);
  A.k_sh = k_strides[1];
  A.v = static_cast<const uint16_t*>(v);
  A.v_st = static_cast<int>(v_strides[0]);
  A.v_sh = v_strides[1];
  A.out = static_cast<uint16_t*>(out);
  A.o_st = out_strides[0];
  A.o_sh = out_strides[1];
  A.cu = cu;
  A.B = static_cast<int>(B);
  A.rows = static_cast<int>(rows);
  A.H = static_cast<int>(Hkv);
  A.G = static_cast<int>(Hq / Hkv);
  A.Hq = static_cast<int>(Hq);
  A.fill = fill;
  A.scale_log2 = scale * kLog2e;
  const int64_t most = max_len < rows ? max_len : rows;
  return launch<false>(A, make_plan(rows, B, Hq, Hkv, most, most), dtype, workspace, workspace_bytes,
                       static_cast<hipStream_t>(stream), what);
}

extern "C" size_t lkv_pages_prefill_attn_workspace_bytes(int64_t rows, int64_t seqs, int64_t Hq, int64_t Hkv,
                                                         int64_t max_new, int64_t max_len) {
  if (rows < 1 || seqs < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || max_new < 0 || max_len < 0) return 0;
  return plan_bytes(make_plan(rows, seqs, Hq, Hkv, max_new < rows ? max_new : rows, max_len), rows, Hq);
}

extern "C" int lkv_pages_prefill_attn(const lkv_pages* p, int64_t layer, const void* q, const int64_t* q_strides,
                                      int64_t rows, int64_t Hq, const int32_t* cu, int64_t max_new, int64_t max_len,
                                      float scale, void* out, const int64_t* out_strides, int fill, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  const char* what = "pages_prefill_attn";
  if (int rc = check_pages(p, what)) return rc;
  LKV_REQUIRE(layer >= 0 && layer < p->layers, "%s: layer %lld of %lld", what, (long long)layer, (long long)p->layers);
  if (int rc = check_queries(rows, Hq, p->kv_heads, cu, what)) return rc;
  LKV_REQUIRE(max_new >= 0 && max_len >= 0 && max_len <= p->width * p->page_size,
              "%s: max_new=%lld, max_len=%lld outside sequences of up to %lld tokens", what, (long long)max_new,
              (long long)max_len, (long long)(p->width * p->page_size));
  if (rows == 0) return LKV_OK;
  if (int rc = check_rows(q, q_strides, what, "q")) return rc;
  if (int rc = check_rows(out, out_strides, what, "out")) return rc;
  Args A{};
  A.q = static_cast<const uint16_t*>(q);
  A.q_st = q_strides[0];
  A.q_sh = q_strides[1];
  A.out = static_cast<uint16_t*>(out);
  A.o_st = out_strides[0];
  A.o_sh = out_strides[1];
  A.cu = cu;
  A.B = static_cast<int>(p->seqs);
  A.rows = static_cast<int>(rows);
  A.st = device_pages(p);
  A.kv = A.st.pool + layer * p->pages * 2 * p->kv_heads * p->page_size * kD;
  A.H = static_cast<int>(p->kv_heads);
  A.G = static_cast<int>(Hq / p->kv_heads);
  A.Hq = static_cast<int>(Hq);
  A.fill = fill;
  A.scale_log2 = scale * kLog2e;
  return launch<true>(A, make_plan(rows, p->seqs, Hq, p->kv_heads, max_new < rows ? max_new : rows, max_len), p->dtype,
                      workspace, workspace_bytes, static_cast<hipStream_t>(stream), what);
}
