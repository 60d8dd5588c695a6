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
// A wave's 32 products a block are in two stretches of 16 with vector work between them: scores of the next block beside
// the exponentials of this one, values of this one beside the next one's offsets and the staging.
//
// What bounds it: two waves per SIMD (240 registers each); per block and wave 1024 cycles of products and about 170 vector
// instructions (4.5 to 6 cycles each, 12 an exponential, with two waves), 3100 cycles for both waves.  Two exponentials,
// four other instructions and an LDS read beside a product take 47 cycles by themselves, a product alone 32.  4096 tokens,
// 32/8 heads: 139-147 us (935-985 TFLOP/s; the library's fp16 product of 8192^3 1069; matrix units busy 54 % of the
// cycles, vector units 59 %, LDS 36 %), chunks of 4 x 512 over 8192 tokens 245 us (1086 TFLOP/s).  Measured on the way:
// products and softmax one after the other 167 us; half of the waves a phase behind, with a barrier a phase 158 us; the
// interleaving with the exponentials left to the compiler 160 us (they move behind the staging); staging without branches,
// workgroups that stay and the exponentials held in place 147 us; output rows through LDS 143 us; staging without bank
// conflicts 139-142 us, chunks 255 to 245 us.  No faster: operands 5 or 6 products ahead, a third key buffer, no running
// maximum (the sum of weights as the check), exponentials moved beside the value products.  What is left outside the blocks
// is a piece's start (10-13 k cycles: lengths, queries, first blocks) and end (4.4 k), 2 a workgroup.
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
constexpr int kXcds = 8;

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
struct PrefillArgs {
  Store st;
  Rows r;
  int tiles;   // column tiles per (sequence, kv head)
  int chunk, splits;
  int items;   // (sequence, kv head) pairs
  int total;   // items * tiles * splits pieces of work
  float* part_o;
  float* part_ml;
};

template <int DT>
__global__ __launch_bounds__(kThr, 1) void prefill_kernel(PrefillArgs P) {
  __shared__ __align__(16) uint16_t smem[2 * kKBuf + 2 * kVBuf];
  uint16_t* const sK = smem;
  uint16_t* const sV = smem + 2 * kKBuf;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c32 = lane & 31, hf = lane >> 5;
  const Store& st = P.st;
  const Rows& r = P.r;

  // ---- staging: waves 0-3 keys (token kk, 32 dims), waves 4-7 values (dim vd, half of its tokens), 16 neighbouring lanes
  // 16 rows, so that their writes fall in distinct banks (4096-token prompt 2-4 % fewer cycles): 2 x 16 bytes of codes
  // a thread, w0 and w1; 16-byte piece p of its four in LDS is dword p of each.  A piece of a key row is then dims
  // 32 part + 4 p + i and 16 + that, and one of a value row tokens 16 p + 4 vh + i and 8 + that: the order of the query
  // operand below, and of a lane's weights.
  const bool key_thr = wave < 4;
  const int kk = 16 * wave + (lane & 15), part = lane >> 4;
  const int vd = 32 * (wave - 4) + 16 * (lane >> 5) + (lane & 15), vh = (lane >> 4) & 1;
  const int src_off = key_thr ? kk * kD + 32 * part : vd * kBlk + 16 * vh;
  const int src2 = key_thr ? 16 : 32;  // the second 16 bytes
  uint16_t* const dst = key_thr ? sK + kk * kKRow + 64 * (part >> 1) + 8 * (part & 1) : sV + vd * kVRow + 8 * vh;
  const int dst_buf = key_thr ? kKBuf : kVBuf;
  const int off = key_thr ? 1 : 0;  // keys are staged a tile further ahead than values
  const uint16_t* const krow = sK + c32 * kKRow + 8 * hf;
  const uint16_t* const vrow = sV + c32 * kVRow + 8 * hf;

  // The workgroups stay and take their pieces of work in turn, the longest first and the order reversed in every second
  // round, so that each gets as much.  Workgroups go to the XCDs round-robin, and the column tiles of one (sequence, kv
  // head) read the same blocks: where the numbers allow it they are all taken on one XCD.
  const int G = r.G;
  const int lanes = gridDim.x % kXcds == 0 && P.items % kXcds == 0 ? kXcds : 1;  // (XCDs apart or not)
  const int width = static_cast<int>(gridDim.x) / lanes;
  const int mine = static_cast<int>(blockIdx.x) / lanes, xcd = static_cast<int>(blockIdx.x) % lanes;
  const int per_lane = P.total / lanes, item_step = P.items / lanes;
#pragma unroll 1
  for (int round = 0; round * width < per_lane; ++round) {
    const int pos = round * width + ((round & 1) ? width - 1 - mine : mine);
    if (pos >= per_lane) continue;  // uniform
    // (divisions leave uniform values in vector registers: made scalar again)
    const int piece = __builtin_amdgcn_readfirstlane(pos / item_step);
    const int item = (pos - piece * item_step) * lanes + xcd;
    const int tile = P.tiles - 1 - __builtin_amdgcn_readfirstlane(piece / P.splits);
    const int split = piece - (P.tiles - 1 - tile) * P.splits;
    const int b = __builtin_amdgcn_readfirstlane(item / st.Hkv), h = item - b * st.Hkv;
    const int len = held_tokens(r.lens[b], r.max_len);
    const int qlen = min(r.q_lens ? min(max(r.q_lens[b], 0), r.S) : r.S, len);
    const int nfull = len / kBlk;
    const int64_t bh = static_cast<int64_t>(b) * st.Hkv + h;
    const int col0 = tile * kCols;
    const int q_first = __builtin_amdgcn_readfirstlane(col0 / G);
    // blocks [blk0, blk1): what the piece's last column sees, of the split's; nf of them finished
    const int last = min(__builtin_amdgcn_readfirstlane((col0 + kCols - 1) / G), qlen - 1);  // its last query
    const int kend = last >= q_first ? len - qlen + last + 1 : 0;
    const int blk0 = split * P.chunk;
    const int blk1 = min(blk0 + P.chunk, (kend + kBlk - 1) / kBlk);
    const int nf = max(min(blk1, nfull) - blk0, 0);
    const bool rest = blk1 > blk0 && blk1 > nfull;  // the unfinished block is the last of them

    // ---- loads that depend on nothing else, all on their way together
    const uint8_t* const src = (key_thr ? st.k_codes : st.v_codes) + (bh * st.blocks + blk0) * kBlkBytes + src_off;
    const float* const scales = st.scales + 2 * (bh * st.blocks + blk0);
    u32x4 w0, w1;
    auto load_tile = [&](int t) {  // (past the last: the last again, staged where nothing reads it)
      const uint8_t* p = src + static_cast<int64_t>(min(t, nf - 1)) * kBlkBytes;
      w0 = *reinterpret_cast<const u32x4*>(p);
      w1 = *reinterpret_cast<const u32x4*>(p + src2);
    };
    auto load_scales = [&](int t) { return *reinterpret_cast<const float2*>(scales + 2 * min(t, nf - 1)); };
    auto stage_piece = [&](int t, int p) {
      *reinterpret_cast<f16x8*>(dst + (t & 1) * dst_buf + 16 * p) = codes8h(w0[p], w1[p]);
    };
    float2 scale = float2{1.f, 1.f}, scale0 = scale;
    u32x4 x0, x1;
    if (nf) {
      load_tile(off);
      x0 = w0;
      x1 = w1;
      load_tile(0);
      scale0 = load_scales(0);
      scale = load_scales(1);
    }
    // ---- the lane's column: query qs, head qh
    const int col = col0 + 32 * wave + c32, qs = col / G, qh = col - qs * G;
    const bool ok = col < r.cols && qs < qlen;
    const int lim = ok ? len - qlen + qs + 1 : 0x7fffffff;  // tokens it sees
    f16x8 qf[8];  // B: step kb: dims 64 (kb / 4) + 32 hf + 4 (kb % 4) + i and 16 + that
    {
      const int64_t at = b * r.q_sb + static_cast<int64_t>(h * G + qh) * r.q_sh + qs * r.q_ss + 32 * hf;
#pragma unroll
      for (int k = 0; k < 8; ++k) qf[k] = f16x8{};
      if (ok) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const f16x8 x[4] = {load_q8<DT>(r.q, at + 64 * k), load_q8<DT>(r.q, at + 64 * k + 8),
                              load_q8<DT>(r.q, at + 64 * k + 16), load_q8<DT>(r.q, at + 64 * k + 24)};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f16x8 lo = x[j >> 1], hi = x[2 + (j >> 1)];
            qf[4 * k + j] = (j & 1) ? __builtin_shufflevector(lo, hi, 4, 5, 6, 7, 12, 13, 14, 15)
                                    : __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 8, 9, 10, 11);
          }
        }
      }
    }
    // tokens that every column of the wave sees
    const int wq = __builtin_amdgcn_readfirstlane((col0 + 32 * wave) / G);
    const int lim_min = wq < qlen ? len - qlen + wq + 1 : 0x7fffffff;

    float m = ok ? -INFINITY : 0.f, l = 0.f;  // a column that is no row keeps offset 0 over zero scores
    f32x16 o[4];  // dims 32 db + 8 (i / 4) + 4 hf + i % 4
#pragma unroll
    for (int db = 0; db < 4; ++db) o[db] = f32x16{};
    f32x16 sc[2];  // scores of tokens 32 kt + 8 (i / 4) + 4 hf + i % 4
    float s[32];   // log2 weights of the present tile, relative to m
    u32x4 pf[4];   // its weights
    constexpr int kAhead = 4;  // operands on their way from LDS
    f16x8 fr[kAhead];
    // operand i of the 16 score products (tile t's keys) and of the 16 value products
    auto key_op = [&](int i, int t) {
      return *reinterpret_cast<const f16x8*>(krow + (t & 1) * kKBuf + 32 * (i & 1) * kKRow + 16 * (i >> 1));
    };
    auto value_op = [&](int i, int t) {
      return *reinterpret_cast<const f16x8*>(vrow + (t & 1) * kVBuf + 32 * (i & 3) * kVRow + 16 * (i >> 2));
    };
    // a tile's factors: key scale * scale * log2(e), log2(value scale), 1 / value scale
    float kc = r.scale_log2, lv = 0.f, iv = 1.f;
    auto factors = [&](const float2& x) {
      const float vs = fmaxf(x.y, kMinScale);
      kc = r.scale_log2 * x.x;
      lv = __log2f(vs);
      iv = __builtin_amdgcn_rcpf(vs);
    };
    auto score_products = [&](int t) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i & 1] = mfma32(key_op(i, t), qf[i >> 1], i < 2 ? f32x16{} : sc[i & 1]);
    };
    // masks and a new offset, where a column of the wave needs one
    auto general = [&](int t) {
      const int left = lim - (blk0 + t) * kBlk - 4 * hf;
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float x = fmaf(sc[e >> 4][e & 15], kc, lv);
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
    float ps[2];
    auto weights = [&](int i) {
      const float a = exp2_(s[2 * i]), c = exp2_(s[2 * i + 1]);
      ps[0] += a;
      ps[1] += c;
      uint32_t u = pk2(a, c);
      __asm__ volatile("" : "+v"(u));  // (no instruction: keeps the work beside the product that it stands next to)
      pf[i >> 2][i & 3] = u;
    };

    // ---- tile 0 (and the keys of tile 1)
    __syncthreads();  // the buffers are free
    if (nf) {
#pragma unroll
      for (int p = 0; p < 4; ++p) stage_piece(0, p);
      if (key_thr) {
        w0 = x0;
        w1 = x1;
#pragma unroll
        for (int p = 0; p < 4; ++p) stage_piece(1, p);
      }
      load_tile(1 + off);
      factors(scale0);
    }
    __syncthreads();
    if (nf) {
      score_products(0);
      general(0);
    }
    __syncthreads();  // (the keys of tile 0 are overwritten next)
    // ---- A tile is two stretches of 16 products, each with vector work between them: the scores of tile t + 1 beside
    // the weights of tile t, then the values of tile t beside the offsets of tile t + 1 and the staging of the next
    // tiles.  Keys and values have two buffers: what a tile overwrites was last read in the tile before.  (Past the last
    // tile the scores are of what lies in LDS, unused.)
#pragma unroll 1
    for (int t = 0; t < nf; ++t) {
      ps[0] = ps[1] = 0.f;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) fr[i] = key_op(i, t + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sc[i & 1] = mfma32(fr[i % kAhead], qf[i >> 1], i < 2 ? f32x16{} : sc[i & 1]);
        fr[i % kAhead] = i + kAhead < 16 ? key_op(i + kAhead, t + 1) : value_op(i + kAhead - 16, t);
        weights(i);
        __builtin_amdgcn_sched_barrier(0);
      }
      l = fmaf(ps[0] + ps[1], iv, l);
      factors(scale);
      const float base = lv - m;
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        o[i & 3] = mfma32(fr[i % kAhead], __builtin_bit_cast(f16x8, pf[i >> 2]), o[i & 3]);
        if (i + kAhead < 16) fr[i % kAhead] = value_op(i + kAhead, t);
        if ((i & 3) == 0) stage_piece(t + 1 + off, i >> 2);
        s[2 * i] = fmaf(sc[i >> 3][2 * i & 15], kc, base);
        s[2 * i + 1] = fmaf(sc[i >> 3][(2 * i + 1) & 15], kc, base);
        mx = fmaxf(fmaxf(mx, s[2 * i]), s[2 * i + 1]);
      }
      load_tile(t + 2 + off);
      scale = load_scales(t + 2);
      if (t + 1 < nf && ((blk0 + t + 2) * kBlk > lim_min || wave_ballot(mx > kMaxWeight) != 0)) general(t + 1);  // uniform
      __syncthreads();
    }
    // ---- the unfinished block: fp16 as it is
    if (rest) {
      const uint16_t* p = tail_ptr(st, !key_thr, bh, blk0 + nf) + src_off;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint2 a = *reinterpret_cast<const uint2*>(p + 4 * k), c = *reinterpret_cast<const uint2*>(p + src2 + 4 * k);
        *reinterpret_cast<u32x4*>(dst + 16 * k) = u32x4{a.x, a.y, c.x, c.y};
      }
      __syncthreads();
      score_products(0);
      kc = r.scale_log2;
      lv = 0.f;
      general(nf);
      ps[0] = ps[1] = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) weights(i);
      l += ps[0] + ps[1];
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i & 3] = mfma32(value_op(i, 0), __builtin_bit_cast(f16x8, pf[i >> 2]), o[i & 3]);
    }

    // (what follows from the lane is computed again here, from a copy: it needs no registers before)
    int out_lane = tid & 63;
    __asm__ volatile("" : "+v"(out_lane));
    const int ox = out_lane & 31, oh = out_lane >> 5;
    const int out_col = col0 + 32 * wave + ox;
    const int out_q = out_col / G, out_h = out_col - out_q * G;
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
    if (P.splits == 1) {
      const bool some = ok && l != 0.f;
      const float inv = some ? 1.f / l : 0.f;
      const int64_t at = b * r.o_sb + static_cast<int64_t>(h * G + out_h) * r.o_sh + out_q * r.o_ss;
      if constexpr (DT == LKV_DTYPE_F32) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int db = 0; db < 2; ++db)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              f32x4 x;
#pragma unroll
              for (int i = 0; i < 4; ++i) x[i] = some ? o[2 * half + db][4 * k + i] * inv : 0.f;
              *reinterpret_cast<f32x4*>(mine_row + 4 * (32 * db + 8 * k + 4 * oh)) = x;
            }
          out_rows(at + 64 * half, out_col < r.cols, [&](int64_t to, const u32x4& v) {
            *reinterpret_cast<u32x4*>(static_cast<float*>(r.out) + to + 4 * (out_lane & 15)) = v;
          });
        }
      } else {
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = some ? o[db][4 * k + i] * inv : 0.f;
            store4<DT>(mine_row, 32 * db + 8 * k + 4 * oh, x[0], x[1], x[2], x[3]);
          }
        out_rows(at, out_col < r.cols, [&](int64_t to, const u32x4& v) {
          *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(r.out) + to + 8 * (out_lane & 15)) = v;
        });
      }
    } else {
      const int64_t at = (bh * r.cols + out_col) * P.splits + split;
      const bool some = ok && blk1 > blk0;
      if (oh == 0 && out_col < r.cols)
        *reinterpret_cast<float2*>(P.part_ml + 2 * at) = some ? part_record(m, l) : part_record(-INFINITY, 0.f);
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
          *reinterpret_cast<u32x4*>(P.part_o + to + 4 * (out_lane & 15)) = v;
        });
      }
    }
  }
}

}  // namespace

int launch_prefill(const Store& store, const Rows& r, const Plan& p, int dtype, int64_t B, float* part_o,
                   float* part_ml, hipStream_t stream) {
  const int64_t items = B * store.Hkv, total = items * p.groups * p.splits;
  LKV_REQUIRE(total < (1ll << 30), "kv8_attn: %lld pieces of work", (long long)total);
  const PrefillArgs A{store, r, p.groups, p.chunk, p.splits, static_cast<int>(items), static_cast<int>(total), part_o,
                      part_ml};
  const int64_t cus = device_cu_count();
  const dim3 grid(static_cast<unsigned>(total < cus ? total : cus));
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
