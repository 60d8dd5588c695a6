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
// only when a weight passes 2^15 (bf16: 2^-20), so that most tiles need no max over lanes and no rescale.
//
// A masked token has weight 0, but 0 times an infinite or NaN value is not 0.  Where a row ends up with such a number its
// workgroup goes through the piece again with care: values that are no numbers count as 0 in the masked tiles' products, and
// a second product counts, of each kind, those that a column sees.
//
// 8 waves, a CU's whole LDS: a row is staged once for 256 columns, and 239 registers (256 over pages) hold a wave's queries, its
// sums and both operands on their way.  Bound by the products (54 % of the SIMDs' cycles over a prompt of 8192) and the vector work beside them
// (52 %): 3480 cycles a tile for the two waves of a SIMD, 2048 of them products, and 12 thousand to begin and end a piece.
// 32/8 heads: a prompt of 8192 tokens 496-606 us by card, 907-1109 TFLOP/s (1.96 GHz under that load where it takes 530; the
// library's product of 8192^3 reached 1241); 4 x 512 queries over 8192 tokens 260-312 us, up to 1030 TFLOP/s; 16 prompts to 1201
// tokens 109-130 us.  Two workgroups a CU of 4 waves and 64-token tiles: 580 where it took 523.
#include "pages_common.h"

namespace lkv {
namespace pages {
namespace {

constexpr int kKRow = kD + 8;   // 16-bit numbers of a staged key row: 16 rows' 16-byte reads fall in distinct banks
constexpr int kVRow = kD + 32;  // and of a value row: the transposing read's 4 rows of 64 bytes do
// A workgroup of W waves: 8 (one a CU), or 4 (two a CU).
template <int W>
struct Shape {
  static constexpr int kPerCu = 8 / W;
  static constexpr int kThr = 64 * W;
  static constexpr int kCols = 32 * W;     // columns
  static constexpr int kTile = 8 * W;      // tokens of a tile: a wave stages 8 rows
  static constexpr int kSub = kTile / 32;  // products along its tokens
  static constexpr int kProducts = 8 * kSub;             // of its scores, and of its values
  static constexpr int kFirst = kProducts * 3 / 4;       // pairs of weights beside the score products, the others beside the
                                                         // values (all beside the scores: 525 us over 8192 tokens, so 517)
  static constexpr int kKBuf = kTile * kKRow, kVBuf = kTile * kVRow;
  static constexpr int kLeast = 6 * kPerCu;  // fewest tiles of a part of the longest piece
};
constexpr int kXcds = 8;
constexpr int kMostCuts = 32;
constexpr int kPlan = 64;         // pieces of a workgroup that are found at once
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
  uint32_t q_st, q_sh;
  uint16_t* out;
  uint32_t o_st, o_sh;
  const int* cu;
  int B, rows;         // sequences, packed rows
  Pages st;            // PAGED: the store, and the layer's pages
  const uint16_t* kv;
  int H, G, Hq;
  int splits;          // most parts of a piece, 1: none is cut
  int fill;
  uint32_t g_mul;      // x / G = x * g_mul >> g_shift for x below 2^31
  int g_shift;
  int g_small, g_big;  // for x below G + 32: (x * g_small >> 16) + (x >= g_big), g_small 0 from G = 32 on, g_big G then
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

__device__ __forceinline__ int by_heads(const Args& P, int x) {
  return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(x)) * P.g_mul >> P.g_shift);
}

// Column tiles of sequence b with more than x tokens to read, of tiles with m rows in all and q of them queries of the last
// of len tokens.
template <int W>
__device__ __forceinline__ int tiles_over(int x, int len, int m, int G) {
  constexpr int kCols = Shape<W>::kCols;
  const int q = min(m, len), all = (m * G + kCols - 1) / kCols;
  const int y = x - (len - q);
  const int under = y >= q ? all : y <= 0 ? 0 : min(all, y * G / kCols);
  return x < 0 ? all : all - under;
}
// Sums over a wave by lane permutes of the vector unit (no LDS round trips: a piece is found with several of them).
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ int moved(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true);
}
__device__ __forceinline__ int wave_prefix(int v) {  // inclusive
  v += moved<0x111>(v);       // row_shr 1, 2, 4, 8
  v += moved<0x112>(v);
  v += moved<0x114>(v);
  v += moved<0x118>(v);
  v += moved<0x142, 0xA>(v);  // row_bcast 15, 31
  v += moved<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_prefix(v), 63); }

// A column tile of T tiles of tokens is j + 1 = ceil(T / chunk) parts (at most `cuts`) of ceil(T / (j + 1)) tiles at most,
// which are more than x < chunk where T > x (j + 1).  Parts of more than x tiles, of all column tiles (x = -1: all parts), are
// then the sum over j of (j + 1) times the tiles with max(j chunk, x (j + 1)) < T <= (j + 1) chunk: with N(y) the tiles with T > y,
//   sum over j of (j + 1) N(max(j chunk, x (j + 1))) - sum over j of j N(j chunk),
// the second the same for all x (`less`).  By the lanes of a wave, a (sequence, j) each.
template <int W>
__device__ __forceinline__ int parts_over(int x, const int* s_len, const int* s_rows, int B, int G, int cuts, int chunk,
                                          int less) {
  constexpr int kTile = Shape<W>::kTile;
  int n = 0;
  const float by = 1.f / cuts;
  for (int i = lane_prefix(~0ull); i < B * cuts; i += 64) {
    const int b = static_cast<int>((i + 0.5f) * by), j = i - b * cuts;  // (exact: i is below 2^18)
    n += (j + 1) * tiles_over<W>(max(j ? j * chunk : -1, x * (j + 1)) * kTile, s_len[b], s_rows[b], G);
  }
  return wave_total(n) - less;
}
template <int W>
__device__ __forceinline__ int parts_less(const int* s_len, const int* s_rows, int B, int G, int cuts, int chunk) {
  int n = 0;
  const float by = 1.f / cuts;
  for (int i = lane_prefix(~0ull); i < B * cuts; i += 64) {
    const int b = static_cast<int>((i + 0.5f) * by), j = i - b * cuts;
    if (j) n += j * tiles_over<W>(j * chunk * Shape<W>::kTile, s_len[b], s_rows[b], G);
  }
  return wave_total(n);
}
// The tiles of the piece-th longest part (from 0), and how many are longer.
template <int W>
__device__ __forceinline__ int part_at(int piece, const int* s_len, const int* s_rows, int B, int G, int longest, int cuts,
                                       int chunk, int less, int& over) {
  int lo = -1, hi = min((longest + Shape<W>::kTile - 1) / Shape<W>::kTile, chunk);
  over = 0;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    const int n = parts_over<W>(mid, s_len, s_rows, B, G, cuts, chunk, less);
    if (n > piece) {
      lo = mid;
    } else {
      hi = mid;
      over = n;
    }
  }
  return hi;
}

// Goes through the workgroup's pieces.  CARE: those that the first time marked in s_again, with care for values that are no
// numbers.  Returns whether any is to be gone through again.
template <int DT, bool PAGED, int W, bool CARE>
__device__ __forceinline__ int go_through(const Args& P, uint16_t* smem, const int* s_len, const int* s_rows,
                                           const int* s_first, int4* s_plan, uint32_t* s_again, int wave, int longest,
                                           int pieces, int cuts, int chunk, int less) {
  using S = Shape<W>;
  constexpr int kWaves = W, kCols = S::kCols, kTile = S::kTile, kSub = S::kSub, kProducts = S::kProducts, kFirst = S::kFirst;
  constexpr int kKBuf = S::kKBuf, kVBuf = S::kVBuf;
  uint16_t* const sK = smem;
  uint16_t* const sV = smem + 2 * kKBuf;
  int lane = lane_prefix(~0ull);
  if (CARE) __asm__ volatile("" : "+v"(lane));  // (what follows from it is not kept from the first time)
  const int c32 = lane & 31, hf = lane >> 5;
  const int G = P.G;
  int again = 0;

  // ---- staging: thread's rows 8 wave + lane / 16 and 4 further, piece lane % 16 of 16 bytes
  const int srow = lane >> 4, spiece = 8 * (lane & 15);
  const int64_t run = PAGED ? run_numbers(P.st) : 0;
  const int k_st = PAGED ? kD : P.k_st, v_st = PAGED ? kD : P.v_st;
  const int koff[2] = {2 * (srow * k_st + spiece), 2 * ((srow + 4) * k_st + spiece)};
  const int voff[2] = {2 * (srow * v_st + spiece), 2 * ((srow + 4) * v_st + spiece)};
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
  const int per_lane = pieces * heads_lane;
  const int every = (per_lane + width - 1) / width;  // rounds, of which the last may have nothing for this workgroup
  auto place_of = [&](int round) { return round * width + ((round & 1) ? width - 1 - own : own); };
  const int rounds = every && place_of(every - 1) >= per_lane ? every - 1 : every;
  // Each begins with another of its pieces, so that not all fetch queries and put rows away at the same time.
  const int shift = rounds ? own % rounds : 0;
  auto turn_of = [&](int round) { return round + shift < rounds ? round + shift : round + shift - rounds; };

  // ---- what the pieces of rounds r .. r + 63 are, found by the waves side by side: the n-th part by the parts' falling length
  auto find_pieces = [&](int r) {
    const ArgsPtr Z = args_again();
    const int n_seqs = Z->B;
    for (int i = wave; i < min(kPlan, rounds - r); i += kWaves) {
      const int pos = place_of(turn_of(r + i));
      const int piece = __builtin_amdgcn_readfirstlane(pos / heads_lane);
      const int h = (pos - piece * heads_lane) * lanes + xcd;
      int over;
      const int size = part_at<W>(piece, s_len, s_rows, n_seqs, G, longest, cuts, chunk, less, over);
      // which of those of its length: by sequence, parts of a tile, and the tile's falling length
      int rank = piece - over, b = 0, tile = 0, split = 0, ns = 1;
      const float by = 1.f / cuts;
      for (int base = 0; base < n_seqs * cuts; base += 64) {
        const int e = base + lane, at_b = static_cast<int>((e + 0.5f) * by), j = e - at_b * cuts;
        int n = 0, high = 0;  // its parts, and its column tiles that are longer
        if (e < n_seqs * cuts) {
          const int len = s_len[at_b], rows = s_rows[at_b], least = j ? j * chunk : -1;
          high = tiles_over<W>(max(least, size * (j + 1)) * kTile, len, rows, G);
          n = (j + 1) * (tiles_over<W>(max(least, (size - 1) * (j + 1)) * kTile, len, rows, G) - high);
        }
        const int sum = wave_prefix(n);
        const uint64_t past = wave_ballot(sum > rank);
        if (past) {
          const int at = __builtin_ctzll(past);
          b = __builtin_amdgcn_readlane(at_b, at);
          ns = __builtin_amdgcn_readlane(j, at) + 1;
          const int mine = rank - __builtin_amdgcn_readlane(sum - n, at), of_tile = mine / ns;
          split = mine - of_tile * ns;
          tile = (s_rows[b] * G + kCols - 1) / kCols - 1 - __builtin_amdgcn_readlane(high, at) - of_tile;
          break;
        }
        rank -= __builtin_amdgcn_readlane(sum, 63);
      }
      // tiles [blk0, blk0 + nt) of 64 tokens: what its last column sees, of the split's
      const int len = s_len[b], rows = s_rows[b], qlen = min(rows, len), col0 = tile * kCols;
      const int last = min(by_heads(P, col0 + kCols - 1), qlen - 1);  // its last query
      const int kend = last >= by_heads(P, col0) ? len - qlen + last + 1 : 0;
      const int all_t = (kend + kTile - 1) / kTile;
      const int part = (all_t + ns - 1) / ns, blk0 = split * part;
      const int nt = max(min(part, all_t - blk0), 0);
      if (lane == 0) {
        s_plan[3 * i] = int4{b, h, split, len};
        s_plan[3 * i + 1] = int4{s_first[b], qlen, rows * G, col0};
        s_plan[3 * i + 2] = int4{blk0, nt, ns, 0};
      }
    }
  };

  struct Piece {
    int b, h, split, len, row0, qlen, cols, col0, blk0, nt, ns, end;  // end: of the tokens that are read
  };
  auto open = [&](int round) {
    if ((round & (kPlan - 1)) == 0) {
      __syncthreads();  // (what it held is read)
      find_pieces(round);
      __syncthreads();
    }
    const int4* f = s_plan + 3 * (round & (kPlan - 1));
    const int4 x = f[0], y = f[1], z = f[2];
    Piece c;
    c.b = __builtin_amdgcn_readfirstlane(x.x);
    c.h = __builtin_amdgcn_readfirstlane(x.y);
    c.split = __builtin_amdgcn_readfirstlane(x.z);
    c.len = __builtin_amdgcn_readfirstlane(x.w);
    c.row0 = __builtin_amdgcn_readfirstlane(y.x);
    c.qlen = __builtin_amdgcn_readfirstlane(y.y);
    c.cols = __builtin_amdgcn_readfirstlane(y.z);
    c.col0 = __builtin_amdgcn_readfirstlane(y.w);
    c.blk0 = __builtin_amdgcn_readfirstlane(z.x);
    c.nt = __builtin_amdgcn_readfirstlane(z.y);
    c.ns = __builtin_amdgcn_readfirstlane(z.z);
    c.end = min(c.len, (c.blk0 + c.nt) * kTile);
    return c;
  };

  // ---- a tile's rows: descriptors of the wave's 8 rows of keys and values
  u32x4 kw[2], vw[2], k1[2];
  // lane i: the page of the wave's rows in tile 64 k + i (past the last tile: the last page, of which nothing is read).
  // (Scalar loads would share their counter with the LDS reads, which then could not be waited for one by one.)
  int pages64 = 0;
  int page1 = 0, page2 = 0;  // pages of the wave's rows in the next tiles
  auto first_of = [&](const Piece& c, int t) { return (c.blk0 + t) * kTile + 8 * wave; };
  auto page_of = [&](const Piece& c, int t) {
    if ((t & 63) == 0) {
      const int e = min(first_of(c, t + lane), c.len - 1) >> P.st.lg;
      pages64 = page_id(P.st, P.st.table[static_cast<int64_t>(c.b) * P.st.width + e]);
    }
    return __builtin_amdgcn_readlane(pages64, t & 63);
  };
  auto load_rows = [&](const Piece& c, int t, u32x4 (&w)[2], const uint16_t* base, int page, int stride, int64_t head,
                       const int (&off)[2]) {
    const int at = first_of(c, t);
    const uint16_t* p = PAGED ? base + (static_cast<int64_t>(page) * 2 * P.H + c.h) * run + (at & (page_size(P.st) - 1)) * kD
                              : base + static_cast<int64_t>(c.row0 + at) * stride + c.h * head;
    // (a row ends within its stride: what lies behind the last one is never asked for)
    const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p), 0, 2 * stride * min(max(c.end - at, 0), 8),
                                                     0x00020000);
#pragma unroll
    for (int j = 0; j < 2; ++j) w[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off[j], 0, 0));
  };
  auto load_k = [&](const Piece& c, int t, u32x4 (&w)[2], int page) {
    load_rows(c, t, w, PAGED ? P.kv : P.k, page, k_st, P.k_sh, koff);
  };
  auto load_v = [&](const Piece& c, int t, int page) {
    load_rows(c, t, vw, PAGED ? P.kv + P.H * run : P.v, page, v_st, P.v_sh, voff);
  };
  auto stage_k = [&](int t, int j) { *reinterpret_cast<u32x4*>(kdst + (t & 1) * kKBuf + 4 * j * kKRow) = kw[j]; };
  auto stage_v = [&](int t, int j) { *reinterpret_cast<u32x4*>(vdst + (t & 1) * kVBuf + 4 * j * kVRow) = vw[j]; };
  // the wave's column r of a piece: query q0 + the first, head the second (r below 32)
  struct Cols {
    int q0, h0;
  };
  auto first_column = [&](const Piece& c) {
    const int x = c.col0 + 32 * wave, q0 = by_heads(P, x);
    return Cols{q0, x - q0 * G};
  };
  auto column = [&](const Cols& w, int r) {
    const int x = w.h0 + r, dq = (x * P.g_small >> 16) + (x >= P.g_big ? 1 : 0);
    return int2{dq, x - dq * G};
  };
  // the wave's own part of LDS, where its query rows and its output rows turn between rows and operands
  constexpr int kOutRow = 272;  // bytes of a row there: 256 and a shift of the banks
  static_assert(32 * kOutRow * kWaves <= 2 * (2 * kKBuf + 2 * kVBuf), "every wave's rows fit");
  char* const turn = reinterpret_cast<char*>(smem) + 32 * kOutRow * wave;
  u32x4 qf[8];  // the wave's query rows, 16 bytes of row 4 j + lane / 16; then B: of the lane's column dims 16 kb + 8 hf ..
  // (A column behind the last row is the last row once more, computed and not put away.)
  auto load_queries = [&](const Piece& c) {
    const Cols w = first_column(c);
    const int end = max(c.qlen * G - 1 - c.col0 - 32 * wave, 0);
    const ArgsPtr Z = args_again();
    const uint32_t q_st = Z->q_st, q_sh = Z->q_sh;
    int r0 = srow;
    __asm__ volatile("" : "+v"(r0));  // (its sums are made where they are used)
    const uint16_t* p = Z->q + static_cast<uint64_t>(c.row0 + min(w.q0, max(c.qlen - 1, 0))) * q_st +
                        static_cast<uint64_t>(c.h * G) * q_sh + spiece;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int2 x = column(w, min(4 * j + r0, end));
      qf[j] = *reinterpret_cast<const u32x4*>(p + (static_cast<uint64_t>(static_cast<uint32_t>(x.x)) * q_st +
                                                   static_cast<uint64_t>(static_cast<uint32_t>(x.y)) * q_sh));
    }
  };
  auto turn_queries = [&]() {
#pragma unroll
    for (int j = 0; j < 8; ++j) *reinterpret_cast<u32x4*>(turn + kOutRow * (4 * j + srow) + 2 * spiece) = qf[j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int kb = 0; kb < 8; ++kb) qf[kb] = *reinterpret_cast<const u32x4*>(turn + kOutRow * c32 + 32 * kb + 16 * hf);
  };
  // the first rows of a piece on their way (the keys of its second tile too), while the last tile of the one before is computed
  // and its rows are put away (asked for after that tile: chunks 1 to 3 % slower)
  auto first_loads = [&](const Piece& c) {
    if (c.nt) {
      int page0 = 0;
      if constexpr (PAGED) {
        page0 = page_of(c, 0);
        page1 = page_of(c, 1);
        page2 = page_of(c, 2);
      }
      load_k(c, 0, kw, page0);
      load_k(c, 1, k1, page1);
      load_v(c, 0, page0);
    }
    load_queries(c);
  };
  if (!rounds) return 0;
  Piece c = open(0);
  if constexpr (!CARE) first_loads(c);
#pragma unroll 1
  for (int round = 0;;) {
    if (CARE) {
      if (round) c = open(round);
      if (!((s_again[(round >> 5) & (kAgain - 1)] >> (round & 31)) & 1)) {  // uniform
        if (++round == rounds) break;
        continue;
      }
      load_queries(c);
    }
    const int len = c.len, qlen = c.qlen, blk0 = c.blk0, nt = c.nt;
    // ---- the lane's column: tokens that it sees; those that every column of the wave sees
    turn_queries();
    const Cols w = first_column(c);
    const int wave_cols = min(qlen * G - c.col0 - 32 * wave, 32);  // columns of the wave that are rows
    const bool works = wave_cols > 0, ok = c32 < wave_cols;
    const int lim = len - qlen + w.q0 + column(w, max(min(c32, wave_cols - 1), 0)).x + 1;
    const int lim_min = len - qlen + w.q0 + 1;

    Piece next = c;
    const bool more = round + 1 < rounds;
    float m, l;
    f32x16 o[4];   // dims 32 db + 8 (i / 4) + 4 hf + i % 4
    f32x16 sc[kSub];  // scores of tokens 32 kt + 8 (i / 4) + 4 hf + i % 4
    float s[16 * kSub];  // log2 weights of the present tile, relative to m
    float ws[2];
    u32x4 pf[2 * kSub];  // its weights
    constexpr int kAhead = 4;  // operands on their way from LDS
    u32x4 fr[kAhead];
    // operand i of the score products (tile t's keys) and of the value products
    auto key_op = [&](int i, int t) {
      return *reinterpret_cast<const u32x4*>(krow + (t & 1) * kKBuf + 32 * (i % kSub) * kKRow + 16 * (i / kSub));
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
      for (int i = 0; i < kProducts; ++i)
        sc[i % kSub] = mfma32<DT>(key_op(i, t), qf[i / kSub], i < kSub ? f32x16{} : sc[i % kSub]);
    };
    // masks and a new offset, where a column of the wave needs one
    auto general = [&](int t) {
      const int left = lim - (blk0 + t) * kTile - 4 * hf;
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16 * kSub; ++e) {
        const float x = sc[e >> 4][e & 15] * kc;
        s[e] = 8 * (e >> 2) + (e & 3) < left ? x : -INFINITY;
        mx = fmaxf(mx, s[e]);
      }
      mx = half_max(mx);
      const float mn = mx - m > max_weight<DT>() ? mx - top_weight<DT>() : m;
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float alpha = exp2_(m - mu);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < 4; ++db) o[db] = o[db] * alpha;
#pragma unroll
      for (int e = 0; e < 16 * kSub; ++e) s[e] -= mu;
    };
    // the same for the first tile, where there are no sums yet
    auto general0 = [&]() {
      float mx = -INFINITY;
      if ((blk0 + 1) * kTile > lim_min) {  // uniform
        const int left = lim - blk0 * kTile - 4 * hf;
#pragma unroll
        for (int e = 0; e < 16 * kSub; ++e) sc[e >> 4][e & 15] = 8 * (e >> 2) + (e & 3) < left ? sc[e >> 4][e & 15] * kc : -INFINITY;
      } else {
#pragma unroll
        for (int kt = 0; kt < kSub; ++kt) sc[kt] = sc[kt] * kc;
      }
#pragma unroll
      for (int e = 0; e < 16 * kSub; ++e) mx = fmaxf(mx, sc[e >> 4][e & 15]);
      mx = half_max(mx);
      m = mx == -INFINITY ? mx : mx - top_weight<DT>();
      const float mu = mx == -INFINITY ? 0.f : m;
#pragma unroll
      for (int e = 0; e < 16 * kSub; ++e) s[e] = sc[e >> 4][e & 15] - mu;
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
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int db = 0; db < 4; ++db) o[db] = f32x16{};
    if constexpr (CARE) {
#pragma unroll 1
      for (int t = 0; t < nt; ++t) {
        int page0 = 0;
        if constexpr (PAGED) page0 = page_of(c, t);
        load_k(c, t, kw, page0);
        load_v(c, t, page0);
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
        for (int i = 0; i < kProducts; ++i) weights(i);
        l += ws[0] + ws[1];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int db = 0; db < 4; ++db) {
          f32x16 count = f32x16{};  // +inf counts 1, -inf 128, NaN both
#pragma unroll
          for (int ks = 0; ks < 2 * kSub; ++ks) {
            const u32x4 raw = value_op(4 * ks + db, 0);
            u32x4 fine, kind, seen;
            int left = lim - (blk0 + t) * kTile - 4 * hf;
            __asm__ volatile("" : "+v"(left));  // (its comparisons are made where they are used)
            no_numbers<DT>(raw, fine, kind);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              // token 16 ks + 4 hf + e % 4 + 8 (e / 4), e = 2 j and 2 j + 1
              const int at = 16 * ks + (2 * j & 3) + 8 * (j >> 1);
              seen[j] = (at < left ? one_bits<DT>() : 0u) | (at + 1 < left ? one_bits<DT>() << 16 : 0u);
            }
            o[db] = mfma32<DT>(fine, pf[ks], o[db]);
            count = mfma32<DT>(kind, seen, count);
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float sum = o[db][i];
            add_counted(count[i], sum);
            o[db][i] = sum;
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
#pragma unroll
        for (int j = 0; j < 2; ++j) *reinterpret_cast<u32x4*>(kdst + kKBuf + 4 * j * kKRow) = k1[j];
        load_v(c, 1, page1);
        load_k(c, 2, kw, page2);
        if constexpr (PAGED) {
          page1 = page2;
          page2 = page_of(c, 3);
        }
      }
      __syncthreads();
      if (works && nt) {
        score_products(0);
        general0();
      }
      __syncthreads();  // (the keys of tile 0 are overwritten next)
      // ---- A tile is two stretches of 16 products, each with vector work between them: the scores of tile t + 1 beside
      // the weights of tile t, then the values of tile t beside the offsets of tile t + 1 and the staging of the next
      // tiles.  Keys and values have two buffers: what a tile overwrites was last read in the tile before.
      auto load_next = [&](int t) {
        load_v(c, t + 2, page1);
        load_k(c, t + 3, kw, page2);
        if constexpr (PAGED) {
          page1 = page2;
          page2 = page_of(c, t + 4);
        }
      };
      if (works) {
#pragma unroll 1
        for (int t = 0; t + 1 < nt; ++t) {
          ws[0] = ws[1] = 0.f;
#pragma unroll
          for (int i = 0; i < kAhead; ++i) fr[i] = key_op(i, t + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < kProducts; ++i) {
            sc[i % kSub] = mfma32<DT>(fr[i % kAhead], qf[i / kSub], i < kSub ? f32x16{} : sc[i % kSub]);
            fr[i % kAhead] = i + kAhead < kProducts ? key_op(i + kAhead, t + 1) : value_op(i + kAhead - kProducts, t);
            if ((i + 1) * kFirst / kProducts > i * kFirst / kProducts) weights(i * kFirst / kProducts);
            __builtin_amdgcn_sched_barrier(0);
          }
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < kProducts; ++i) {
            o[i & 3] = mfma32<DT>(fr[i % kAhead], pf[i >> 2], o[i & 3]);
            if (i + kAhead < kProducts) fr[i % kAhead] = value_op(i + kAhead, t);
            if (i % (kProducts / 4) == 0) {
              const int j = i / (kProducts / 4);
              if (j < 2)
                stage_k(t + 2, j);
              else
                stage_v(t + 1, j - 2);
            }
            // (the last weights: before the products that take them, and before their scores are written over)
            constexpr int kLast = kProducts - kFirst, kBy = 2 * kLast;
            if (i < kBy && (i + 1) * kLast / kBy > i * kLast / kBy) weights(kFirst + i * kLast / kBy);
            s[2 * i] = fmaf(sc[i >> 3][2 * i & 15], kc, -m);
            s[2 * i + 1] = fmaf(sc[i >> 3][(2 * i + 1) & 15], kc, -m);
            mx = fmaxf(fmaxf(mx, s[2 * i]), s[2 * i + 1]);
            __builtin_amdgcn_sched_barrier(0);
          }
          l += ws[0] + ws[1];
          load_next(t);
          if ((blk0 + t + 2) * kTile > lim_min || wave_ballot(mx > max_weight<DT>()) != 0) general(t + 1);  // uniform
          __syncthreads();
        }
      } else {  // no columns: the wave's part of the staging
#pragma unroll 1
        for (int t = 0; t + 1 < nt; ++t) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            stage_k(t + 2, j);
            stage_v(t + 1, j);
          }
          load_next(t);
          __syncthreads();
        }
      }
      if (more) {
        next = open(round + 1);
        first_loads(next);
      }
      if (works && nt) {  // the last tile
        ws[0] = ws[1] = 0.f;
#pragma unroll
        for (int i = 0; i < kProducts; ++i) weights(i);
        l += ws[0] + ws[1];
#pragma unroll
        for (int i = 0; i < kProducts; ++i) o[i & 3] = mfma32<DT>(value_op(i, nt - 1), pf[i >> 2], o[i & 3]);
      }
      __syncthreads();  // the tiles are done with
    }

    if constexpr (!CARE) {  // an infinity or NaN times 0 is NaN, and NaN != 0
      f32x4 odd = f32x4{};
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) odd[i & 3] = fmaf(o[db][i], 0.f, odd[i & 3]);
      if (wave_ballot(ok && (odd[0] + odd[1]) + (odd[2] + odd[3]) != 0.f)) {
        if (lane == 0) atomicOr(&s_again[(round >> 5) & (kAgain - 1)], 1u << (round & 31));
        again = 1;
      }
    }
    const ArgsPtr Z = args_again();
    // (what follows from the lane is computed again here, from a copy: it needs no registers before)
    int out_lane = lane_prefix(~0ull);
    __asm__ volatile("" : "+v"(out_lane));
    const int ox = out_lane & 31, oh = out_lane >> 5;
    // ---- out: a wave's 32 rows through its part of LDS (the tiles are done with), so that a row goes out whole
    l = half_sum(l);
    if constexpr (CARE) __syncthreads();  // (the tiles' last barrier, otherwise)
    char* const mine_row = turn + kOutRow * ox;
    // row 4 j + lane / 16 as a lane puts it away: 16 bytes of it to put(query, head, bytes)
    const Cols first = first_column(c);
    const int ends = c.cols - c.col0 - 32 * wave;
    auto out_rows = [&](int end, auto put) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = 4 * j + (out_lane >> 4);
        const u32x4 v = *reinterpret_cast<const u32x4*>(turn + kOutRow * row + 16 * (out_lane & 15));
        const int2 x = column(first, row);
        if (row < end) put(static_cast<uint32_t>(x.x), static_cast<uint32_t>(x.y), v);
      }
    };
    const int slots = Z->splits;
    if (c.ns == 1) {
      if (slots > 1 && oh == 0 && ox < ends) {  // (a mark for the join: this row is done)
        const int2 x = column(first, ox);
        const int64_t at = static_cast<int64_t>(c.row0 + first.q0 + x.x) * Z->Hq + c.h * G + x.y;
        *reinterpret_cast<float2*>(Z->part_ml + 2 * at * slots) = float2{-INFINITY, -1.f};
      }
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
      uint16_t* const base =
          Z->out + static_cast<uint64_t>(c.row0 + first.q0) * Z->o_st + static_cast<uint64_t>(c.h * G) * Z->o_sh;
      const uint32_t o_st = Z->o_st, o_sh = Z->o_sh;
      out_rows(ends, [&](uint32_t q, uint32_t x, const u32x4& v) {
        *reinterpret_cast<u32x4*>(base + (static_cast<uint64_t>(q) * o_st + static_cast<uint64_t>(x) * o_sh + 8 * (out_lane & 15))) = v;
      });
    } else {
      // (a split without tokens leaves its rows unwritten: its record is empty)
      const int64_t base = (static_cast<int64_t>(c.row0 + first.q0) * Z->Hq + c.h * G) * slots + c.split;
      const uint32_t by_q = Z->Hq * slots, by_h = slots;
      if (oh == 0 && ox < ends) {
        const int2 x = column(first, ox);
        const int64_t at = base + static_cast<int64_t>(x.x) * by_q + static_cast<int64_t>(x.y) * by_h;
        float2* const ml = reinterpret_cast<float2*>(Z->part_ml) + at;
        *ml = ok && nt > 0 ? part_record(m, l) : part_record(-INFINITY, 0.f);
        if (c.split == 0)
          for (int i = c.ns; i < slots; ++i) ml[i] = part_record(-INFINITY, 0.f);
      }
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
        out_rows(nt ? wave_cols : 0, [&](uint32_t q, uint32_t x, const u32x4& v) {
          const int64_t at = base + static_cast<int64_t>(q) * by_q + static_cast<int64_t>(x) * by_h;
          *reinterpret_cast<u32x4*>(Z->part_o + at * kD + 64 * half + 4 * (out_lane & 15)) = v;
        });
      }
    }
    if (!more) break;
    c = next;
    ++round;
  }
  return again;
}

template <int DT, bool PAGED, int W>
__global__ __launch_bounds__(Shape<W>::kThr, 2) void prefill_kernel(Args P) {
  using S = Shape<W>;
  constexpr int kWaves = W, kPerCu = S::kPerCu, kThr = S::kThr, kCols = S::kCols, kTile = S::kTile, kLeast = S::kLeast;
  __shared__ __align__(16) uint16_t smem[2 * S::kKBuf + 2 * S::kVBuf];
  __shared__ int s_len[kMaxSeqs], s_rows[kMaxSeqs], s_first[kMaxSeqs];
  __shared__ int4 s_plan[3 * kPlan];
  __shared__ uint32_t s_again[kAgain];  // pieces to go through again, by round
  __shared__ int s_any;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tid = threadIdx.x, lane = tid & 63;
  const int G = P.G;

  // ---- every sequence's tokens and rows; the longest
  int longest = 0;
  for (int b = tid; b < P.B; b += kThr) {
    const int a = min(max(P.cu[b], 0), P.rows), e = min(max(P.cu[b + 1], a), P.rows);
    s_first[b] = a;
    s_rows[b] = e - a;
    s_len[b] = PAGED ? held(P.st, P.st.lens[b]) : e - a;
  }
  if (tid < kAgain) s_again[tid] = 0;
  if (tid == 0) s_any = 0;
  __syncthreads();
  int pieces = 0;  // column tiles of all sequences
  int low = 0, high = 0;  // their rows
  for (int b = lane; b < P.B; b += 64) {
    longest = max(longest, s_len[b]);
    pieces += tiles_over<W>(-1, s_len[b], s_rows[b], G);
    low += s_rows[b] & 0xffff;
    high += s_rows[b] >> 16;
  }
  // Starts that fall: sequences would lie over each other, and their pieces pass what the launch counted with.  None is taken.
  low = wave_total(low);
  high = wave_total(high) + (low >> 16);
  if (high > P.rows >> 16 || (high == P.rows >> 16 && (low & 0xffff) > (P.rows & 0xffff))) {  // uniform
    __syncthreads();
    for (int b = tid; b < P.B; b += kThr) s_rows[b] = 0;
    __syncthreads();
    pieces = 0;
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) longest = max(longest, __shfl_xor(longest, x));
  longest = __builtin_amdgcn_readfirstlane(longest);
  pieces = wave_total(pieces);

  // ---- into how many parts the longest pieces are cut.  What that takes, in tiles: the longest part, or the workgroups' mean
  // and some of a part (in two rounds what the last of the first and the first of the second take, if that is more), about 4
  // a round for beginning and ending pieces, and writing and joining the parts' rows (a launch is 2.5 tiles' time, 7.6e6 bytes a
  // tile's time are what the card writes and reads again).  All of it was measured with 32/8 heads, where a tile takes 1.8
  // us; the shares of a part, 0.15 and 0.3, and the 5 % by which a cut has to gain are not derived but set by times of chunks over
  // 0.4 to 17 K tokens there.  They choose between divisions that are all right.  The waves look at every eighth number each.
  int cuts = 1, chunk = 1 << 24, less = 0;
  if (P.splits > 1) {
    float work = 0.f;
    int cols = 0;
    for (int b = lane; b < P.B; b += 64) {
      const int len = s_len[b], rows = s_rows[b], q = min(rows, len);
      work += tiles_over<W>(-1, len, rows, G) * (len - 0.5f * q + 0.5f * min(kCols / G, q) + 0.5f * kTile) * (1.f / kTile);
      cols += rows * G;
    }
#pragma unroll
    for (int x = 32; x; x >>= 1) work += __shfl_xor(work, x);
    cols = wave_total(cols);
    const float grid = gridDim.x, mean = work * P.H / grid;
    const int most = (longest + kTile - 1) / kTile;
    for (int k = wave + 1; k <= P.splits; k += kWaves) {
      const int part = (most + k - 1) / k;
      int n = pieces, cut = 0, lost = 0;  // parts in all, column tiles that are cut
      if (k > 1) {
        lost = parts_less<W>(s_len, s_rows, P.B, G, k, part);
        n = parts_over<W>(-1, s_len, s_rows, P.B, G, k, part, lost);
        for (int b = lane; b < P.B; b += 64) cut += tiles_over<W>(part * kTile, s_len[b], s_rows[b], G);
        cut = wave_total(cut);
      }
      const float items = static_cast<float>(n) * P.H;
      const float load = items <= grid ? part : fmaxf(mean + (items <= 2.f * grid ? 0.15f : 0.3f) * part, part);
      const float part_rows = static_cast<float>(min(cut * kCols, cols)) * (P.H * k);
      const float join = k > 1 ? 2.5f * kPerCu + part_rows * (1040 * kPerCu / 7.6e6f) : 0.f;
      const float around = 4.f * kPerCu * ceilf(items / grid) + join;
      const bool two = items > grid && items <= 2.f * grid;
      if (lane == 0)
        s_plan[k - 1] = int4{__float_as_int(k > 1 && part < kLeast ? INFINITY : (load + around) * (k > 1 ? 1.05f : 1.f)), n,
                             lost, __float_as_int(two ? around : -1.f)};
    }
    __syncthreads();
    // (what those two parts take is only looked for where it could matter)
    int4 mine = int4{__float_as_int(INFINITY), 0, 0, 0};
    if (lane < P.splits) mine = s_plan[lane];
    float best = __int_as_float(mine.w) < 0.f ? __int_as_float(mine.x) : INFINITY;
#pragma unroll
    for (int x = 32; x; x >>= 1) best = fminf(best, __shfl_xor(best, x));
    __syncthreads();
    for (int k = wave + 1; k <= P.splits; k += kWaves) {
      const float takes = __int_as_float(__builtin_amdgcn_readlane(mine.x, k - 1));
      const float around = __int_as_float(__builtin_amdgcn_readlane(mine.w, k - 1));
      if (around < 0.f || takes >= best) continue;
      const int n = __builtin_amdgcn_readlane(mine.y, k - 1), lost = __builtin_amdgcn_readlane(mine.z, k - 1);
      const int nth = min(static_cast<int>(gridDim.x) / P.H, n - 1), part = k > 1 ? (most + k - 1) / k : 1 << 24;
      int over, two = 0;
#pragma unroll 1
      for (int i = max(nth - 1, 0); i <= nth; ++i)
        two += part_at<W>(i, s_len, s_rows, P.B, G, longest, k, part, lost, over);
      if (lane == 0) s_plan[k - 1].x = __float_as_int(fmaxf(takes, (two + around) * (k > 1 ? 1.05f : 1.f)));
    }
    __syncthreads();
    best = lane < P.splits ? __int_as_float(s_plan[lane].x) : INFINITY;
    float least = best;
#pragma unroll
    for (int x = 32; x; x >>= 1) least = fminf(least, __shfl_xor(least, x));
    const int at = __builtin_ctzll(wave_ballot(best == least));
    cuts = at + 1;
    pieces = __builtin_amdgcn_readlane(mine.y, at);
    less = __builtin_amdgcn_readlane(mine.z, at);
    cuts = __builtin_amdgcn_readfirstlane(cuts);
    if (cuts > 1) chunk = (most + cuts - 1) / cuts;
  }

  const int again = go_through<DT, PAGED, W, false>(P, smem, s_len, s_rows, s_first, s_plan, s_again, wave, longest, pieces,
                                                    cuts, chunk, less);
  if (again && lane == 0) s_any = 1;
  __syncthreads();
  if (s_any) {
    go_through<DT, PAGED, W, true>(P, smem, s_len, s_rows, s_first, s_plan, s_again, wave, longest, pieces, cuts, chunk,
                                   less);
  }

  // ---- rows of no sequence
  const ArgsPtr Z = args_again();
  if (Z->fill) {
    const int a = min(max(Z->cu[0], 0), Z->rows), e = min(max(Z->cu[Z->B], a), Z->rows);
    const int64_t per = static_cast<int64_t>(Z->Hq) * (kD / 8), n = (a + Z->rows - e) * per;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThr;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThr + 64 * wave + lane_prefix(~0ull); i < n; i += step) {
      const int64_t r = i / per, x = i - r * per;
      const int64_t row = r < a ? r : r - a + e;
      *reinterpret_cast<u32x4*>(Z->out + row * Z->o_st + x / (kD / 8) * Z->o_sh + 8 * (x % (kD / 8))) = u32x4{};
    }
  }
}

struct Plan {
  int waves;       // of a workgroup
  int64_t pieces;  // most column tiles of a kv head, over all sequences
  int splits;      // parts that a piece may be cut into (the kernel decides, by the lengths)
};

// enough: so many pieces a CU are shared out evenly enough as they are.
template <int W>
Plan plan_for(int64_t rows, int64_t B, int64_t Hq, int64_t Hkv, int64_t max_new, int64_t max_len, float enough) {
  using S = Shape<W>;
  const int64_t G = Hq / Hkv;
  const int64_t each = B * ((max_new * G + S::kCols - 1) / S::kCols), packed = rows * G / S::kCols + B;
  Plan p;
  p.waves = W;
  p.pieces = each < packed ? each : packed;
  p.pieces = p.pieces < 1 ? 1 : p.pieces;
  const int64_t cus = device_cu_count() * S::kPerCu, tiles = (max_len + S::kTile - 1) / S::kTile, work = p.pieces * Hkv;
  int64_t splits = work >= enough * cus ? 1 : (3 * cus + work - 1) / work;
  splits = splits > tiles / S::kLeast ? tiles / S::kLeast : splits;
  p.splits = static_cast<int>(splits < 1 ? 1 : splits > kMostCuts ? kMostCuts : splits);
  return p;
}
// Whole prompts.  Two workgroups of 4 waves a CU up to 256 tokens, where beginning and ending pieces is most of the work and one
// fills the other's waits, and up to 2048 tokens where 8 waves would have no more than a piece for each CU (half as large, twice
// as many are shared out more evenly).  With 8 waves, and with 4, 32/8 heads: 64 prompts to 150 tokens 30.2 and 24.5 us, 64 x 64
// 24.9 and 22.2, 1 x 512 22.8 and 20.8, 900, 300 and 200 tokens 32.7 and 30.3, 1 x 2048 65.3 and 65; but 16 x 512 63 and 65, 1 x
// 8192 525 and 605: every row of keys and values is staged twice as often.  From 0.75 pieces a workgroup on (4 waves: 0.6) none
// is cut (1 x 2048 tokens, a piece a CU: cutting the longer ones costs as much in rows to join as it gains).
Plan packed_plan(int64_t rows, int64_t B, int64_t Hq, int64_t Hkv, int64_t max_len) {
  const int64_t most = max_len < rows ? max_len : rows;
  const Plan p = plan_for<8>(rows, B, Hq, Hkv, most, most, 0.75f);
  const bool four = most <= 256 || (most <= 2048 && p.pieces * Hkv <= device_cu_count());
  return four ? plan_for<4>(rows, B, Hq, Hkv, most, most, 0.6f) : p;
}
// Over pages, from two pieces a CU on none is cut (the launch that joins costs 5 us where none is).  Chunks to 512 over 1.6-8 K
// tokens of 4 sequences, 0.8 pieces a CU: 268 us as they are, 230 in two parts taken by the length of their tiles, 168 in three
// by their own length; 12 sequences of 0.4-17 K, 1.5 pieces a CU: 458 and 301 us.
Plan pages_plan(int64_t rows, int64_t B, int64_t Hq, int64_t Hkv, int64_t max_new, int64_t max_len) {
  return plan_for<8>(rows, B, Hq, Hkv, max_new < rows ? max_new : rows, max_len, 2.f);
}

size_t plan_bytes(const Plan& p, int64_t rows, int64_t Hq) {
  return p.splits == 1 ? 0 : static_cast<size_t>(rows * Hq) * p.splits * (kD + 2) * 4;
}

template <bool PAGED, int W>
int launch_shape(const Args& A, const Plan& p, int dtype, hipStream_t s, const char* what) {
  using S = Shape<W>;
  const int64_t work = p.pieces * p.splits * A.H, cus = device_cu_count() * S::kPerCu;
  const int64_t most = (static_cast<int64_t>(A.rows) * A.G / S::kCols + A.B) * p.splits * A.H;  // whatever cu holds
  LKV_REQUIRE(most < (1ll << 30), "%s: %lld pieces of work", what, (long long)most);
  const dim3 grid(static_cast<unsigned>(work < cus ? work : cus));
  if (dtype == LKV_DTYPE_F16)
    hipLaunchKernelGGL((prefill_kernel<LKV_DTYPE_F16, PAGED, W>), grid, dim3(S::kThr), 0, s, A);
  else
    hipLaunchKernelGGL((prefill_kernel<LKV_DTYPE_BF16, PAGED, W>), grid, dim3(S::kThr), 0, s, A);
  LKV_LAUNCH_CHECK(what);
  return LKV_OK;
}

template <bool PAGED>
int launch(Args A, const Plan& p, int dtype, void* workspace, size_t workspace_bytes, hipStream_t s, const char* what) {
  const size_t need = plan_bytes(p, A.rows, A.Hq);
  LKV_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && aligned16(workspace))),
              "%s: a 16-byte aligned workspace of %zu bytes required, got %zu", what, need, workspace_bytes);
  A.g_shift = 31;
  while ((1ll << (A.g_shift - 31)) < A.G) ++A.g_shift;
  A.g_mul = static_cast<uint32_t>((1ull << A.g_shift) / A.G + 1);
  A.g_small = A.G < 32 ? 65536 / A.G + 1 : 0;
  A.g_big = A.G < 32 ? 0x7fffffff : A.G;
  A.splits = p.splits;
  A.part_o = static_cast<float*>(workspace);
  A.part_ml = A.part_o + static_cast<size_t>(A.rows) * A.Hq * p.splits * kD;
  int rc;
  if constexpr (PAGED)
    rc = launch_shape<true, 8>(A, p, dtype, s, what);
  else
    rc = p.waves == 4 ? launch_shape<false, 4>(A, p, dtype, s, what) : launch_shape<false, 8>(A, p, dtype, s, what);
  if (rc || p.splits == 1) return rc;
  return launch_join(A.part_o, A.part_ml, static_cast<int64_t>(A.rows) * A.Hq, p.splits, A.Hq, A.out, A.o_st, A.o_sh,
                     dtype, A.cu, A.B, s, what);
}

// So few columns of a kv head that the few-row kernel, whose waves read their rows by themselves, takes them.
bool few(int64_t rows, int64_t Hq, int64_t Hkv, int64_t max_new) {
  return (max_new < rows ? max_new : rows) * (Hq / Hkv) <= 32;
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
  return plan_bytes(packed_plan(rows, B, Hq, Hkv, max_len), rows, Hq);
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
  LKV_REQUIRE(rows == 1 || (k_strides[0] >= kD && v_strides[0] >= kD), "%s: rows of k or v overlap", what);
  Args A{};
  A.q = static_cast<const uint16_t*>(q);
  A.q_st = static_cast<uint32_t>(q_strides[0]);
  A.q_sh = static_cast<uint32_t>(q_strides[1]);
  A.k = static_cast<const uint16_t*>(k);
  A.k_st = rows == 1 ? kD : static_cast<int>(k_strides[0]);
  A.k_sh = k_strides[1];
  A.v = static_cast<const uint16_t*>(v);
  A.v_st = rows == 1 ? kD : static_cast<int>(v_strides[0]);
  A.v_sh = v_strides[1];
  A.out = static_cast<uint16_t*>(out);
  A.o_st = static_cast<uint32_t>(out_strides[0]);
  A.o_sh = static_cast<uint32_t>(out_strides[1]);
  A.cu = cu;
  A.B = static_cast<int>(B);
  A.rows = static_cast<int>(rows);
  A.H = static_cast<int>(Hkv);
  A.G = static_cast<int>(Hq / Hkv);
  A.Hq = static_cast<int>(Hq);
  A.fill = fill;
  A.scale_log2 = scale * kLog2e;
  return launch<false>(A, packed_plan(rows, B, Hq, Hkv, max_len), dtype, workspace, workspace_bytes,
                       static_cast<hipStream_t>(stream), what);
}

extern "C" size_t lkv_pages_prefill_attn_workspace_bytes(int64_t rows, int64_t seqs, int64_t Hq, int64_t Hkv,
                                                         int64_t max_new, int64_t max_len) {
  if (rows < 1 || seqs < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || max_new < 0 || max_len < 0) return 0;
  if (few(rows, Hq, Hkv, max_new)) return few_rows_bytes(rows, seqs, Hq, Hkv, max_len);
  return plan_bytes(pages_plan(rows, seqs, Hq, Hkv, max_new, max_len), rows, Hq);
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
  if (few(rows, Hq, p->kv_heads, max_new))
    return launch_few_rows(p, layer, q, q_strides, rows, Hq, cu, max_len, scale, out, out_strides, fill, workspace,
                           workspace_bytes, static_cast<hipStream_t>(stream), what);
  Args A{};
  A.q = static_cast<const uint16_t*>(q);
  A.q_st = static_cast<uint32_t>(q_strides[0]);
  A.q_sh = static_cast<uint32_t>(q_strides[1]);
  A.out = static_cast<uint16_t*>(out);
  A.o_st = static_cast<uint32_t>(out_strides[0]);
  A.o_sh = static_cast<uint32_t>(out_strides[1]);
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
  return launch<true>(A, pages_plan(rows, p->seqs, Hq, p->kv_heads, max_new, max_len), p->dtype,
                      workspace, workspace_bytes, static_cast<hipStream_t>(stream), what);
}
