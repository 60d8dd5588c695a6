// Page tables of the 16-bit paged KV cache: room for new tokens, forking, compacting, and the rows themselves (store, read).
//
// All bookkeeping lives on the device, so that a step that grows or forks sequences is captured once and replayed.
//   extend    one workgroup: what every sequence needs (new pages, and a copy of a shared last page that is not full),
//             prefix sums over the sequences, the lowest free pages by a scan of refs, who waits where those run out, table
//             and lens.  Then one launch that copies the shared tokens in every layer (nothing to do in most steps).
//   fork      a workgroup per sequence writes its new row to the workspace and counts refs by integer atomics (their order
//             does not matter); a second launch puts the rows in place, since sequences take each other's rows.
//   compact   one workgroup ranks free pages below and used pages from n on; a second launch moves pages and renames
//             table entries.  Pages that move and the places they move to are apart, so that nothing is overwritten early.
//   store     a wave per token.
// Each is a launch or two of 2 to 8 us (latency: a few dependent reads of the tables) but for what is moved: store 90.6 MB read
// and written in 16-17 us (5.4 TB/s), compact 359 MB in 73 us (4.9 TB/s; a device copy reaches 5.13),
// read 268 MB in 39 us (8 sequences of 4096 tokens, 8 heads, pages of 16 or 64: 6.8 TB/s over and over, part of it from the
// last-level cache), 4096 tokens of one in 7.5 us.
#include "pages_common.h"

namespace lkv {
namespace pages {
namespace {

constexpr int kPlanThr = 1024;
constexpr int kThr = 256;

// Exclusive prefix sum over a workgroup of 1024 threads; total is the sum over all of them.
__device__ __forceinline__ int block_prefix(int v, int* s_wave, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // (what s_wave held is read)
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThr / 64; ++w) {
    const int t = s_wave[w];
    before += w < wave ? t : 0;
    total += t;
  }
  return before + x - v;
}

// Four refs from page p on; pages past the pool count as `past`.
__device__ __forceinline__ void refs4(const Pages& st, int p, int past, int (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = p + i < st.pages ? st.refs[p + i] : past;
}

struct ExtendArgs {
  Pages st;
  const int* cu;
  int* free_list;  // [pages]
  int* copies;     // [1 + 3 seqs]: their number, then (from, to, tokens) of each
};

__device__ __forceinline__ int new_tokens(const ExtendArgs& A, int s, int len) {
  const int n = A.cu ? A.cu[s + 1] - A.cu[s] : (len > 0 ? 1 : 0);
  return n > 0 && n <= (A.st.width << A.st.lg) - len ? n : 0;
}

__global__ __launch_bounds__(kPlanThr) void extend_kernel(ExtendArgs A) {
  __shared__ int s_last[kMaxSeqs];       // a shared last page that is not full, or -1
  __shared__ int s_meta[kMaxSeqs];       // 4 * pages held + 2 * whether it waits for another + whether the last one is to be copied
  __shared__ int s_begin[kMaxSeqs + 1];  // pages needed by the sequences before
  __shared__ int s_wave[kPlanThr / 64];
  __shared__ int s_copies;
  const Pages& st = A.st;
  const int tid = threadIdx.x, S = st.seqs, mask = page_size(st) - 1;
  if (tid == 0) s_copies = 0;

  int shared = 0;
  for (int s = tid; s < S; s += kPlanThr) {
    const int len = held(st, st.lens[s]), n = new_tokens(A, s, len);
    const int old = (len + mask) >> st.lg;
    int last = -1;
    if (n > 0 && (len & mask)) {
      last = page_id(st, st.table[static_cast<int64_t>(s) * st.width + (len >> st.lg)]);
      if (st.refs[last] <= 1) last = -1;
    }
    s_last[s] = last;
    s_meta[s] = 4 * old;
    s_begin[s] = ((len + n + mask) >> st.lg) - old;
    shared |= last >= 0 ? 1 : 0;
  }
  shared = __syncthreads_or(shared);
  if (shared) {
    for (int s = tid; s < S; s += kPlanThr) {
      const int last = s_last[s];
      if (last < 0) continue;
      int writers = 0, before = 0;
      for (int t = 0; t < S; ++t) {
        const int same = s_last[t] == last ? 1 : 0;
        writers += same;
        before += t < s ? same : 0;
      }
      if (before || writers != st.refs[last]) {
        s_meta[s] += 1;
        s_begin[s] += 1;
      }
    }
  }
  int total = 0;
  for (int base = 0; base < S; base += kPlanThr) {
    const int s = base + tid;
    const int v = s < S ? s_begin[s] : 0;
    int sum;
    const int at = total + block_prefix(v, s_wave, sum);
    if (s < S) s_begin[s] = at;
    total += sum;
  }
  if (tid == 0) s_begin[S] = total;

  // the lowest free pages, at most as many as are needed
  int found = 0;
  for (int base = 0; base < st.pages && found < total; base += 4 * kPlanThr) {
    const int p = base + 4 * tid;
    int r[4];
    refs4(st, p, 1, r);
    int v = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) v += r[i] <= 0 ? 1 : 0;
    int sum;
    int at = found + block_prefix(v, s_wave, sum);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r[i] <= 0) {
        if (at < total) A.free_list[at] = p + i;
        ++at;
      }
    found += sum;
  }
  const int got = min(found, total);
  __threadfence_block();
  __syncthreads();
  // Pages ran out.  A copy that is not there leaves its sequence on the shared page, so the first of the page, which would go on
  // in it, waits too where that sequence holds more tokens of it than the first does.
  if (got < total && shared) {
    for (int s = tid; s < S; s += kPlanThr) {
      const int last = s_last[s];
      if (last < 0 || (s_meta[s] & 1)) continue;
      const int len = held(st, st.lens[s]);
      for (int t = s + 1; t < S; ++t)
        if (s_last[t] == last && s_begin[t + 1] > got && held(st, st.lens[t]) > len) {
          s_meta[s] += 2;
          break;
        }
    }
    __syncthreads();
  }
  for (int r = tid; r < got; r += kPlanThr) {
    int lo = 0, hi = S;  // the sequence with s_begin[s] <= r < s_begin[s + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_begin[mid] <= r)
        lo = mid;
      else
        hi = mid;
    }
    if (s_begin[lo + 1] > got || (s_meta[lo] & 2)) continue;  // its pages are not all there, or it waits
    const int j = r - s_begin[lo], old = s_meta[lo] >> 2, copy = s_meta[lo] & 1;
    const int page = A.free_list[r];
    st.refs[page] = 1;
    st.table[static_cast<int64_t>(lo) * st.width + old + j - copy] = page;
    if (copy && j == 0) {
      const int from = s_last[lo], c = 3 * atomicAdd(&s_copies, 1);
      atomicSub(&st.refs[from], 1);
      A.copies[1 + c] = from;
      A.copies[2 + c] = page;
      A.copies[3 + c] = held(st, st.lens[lo]) & mask;
    }
  }
  __syncthreads();
  if (tid == 0) A.copies[0] = s_copies;
  for (int s = tid; s < S; s += kPlanThr) {
    const int len = held(st, st.lens[s]);
    const bool fits = (s_begin[s + 1] == s_begin[s] || s_begin[s + 1] <= got) && !(s_meta[s] & 2);
    const int n = fits ? new_tokens(A, s, len) : 0;
    st.lens[s] = len + n;
    st.taken[s] = n;
  }
}

// The first tokens of pages, in every layer: a workgroup takes the rows of one (copy, layer, side, head).
__global__ __launch_bounds__(kThr) void copy_kernel(Pages st, const int* copies) {
  const int per = st.layers * 2 * st.H;
  const int64_t units = static_cast<int64_t>(copies[0]) * per;
  const int64_t run = run_numbers(st), page = page_numbers(st);
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int c = static_cast<int>(u / per), rest = static_cast<int>(u - static_cast<int64_t>(c) * per);
    const int layer = rest / (2 * st.H);
    uint16_t* base = st.pool + static_cast<int64_t>(layer) * st.pages * page + (rest - layer * 2 * st.H) * run;
    const u32x4* from = reinterpret_cast<const u32x4*>(base + copies[1 + 3 * c] * page);
    u32x4* to = reinterpret_cast<u32x4*>(base + copies[2 + 3 * c] * page);
    const int n = copies[3 + 3 * c] * (kD / 8);
    for (int i = threadIdx.x; i < n; i += kThr) to[i] = from[i];
  }
}

struct ForkArgs {
  Pages st;
  const int* parent;
  const int* cut;
  int* rows;  // [seqs][width]
  int* lens;  // [seqs]
};

__device__ __forceinline__ int fork_source(const ForkArgs& A, int s, int& len) {
  const int p = A.parent ? A.parent[s] : s;
  const bool ok = p >= 0 && p < A.st.seqs;
  len = ok ? held(A.st, A.st.lens[p]) : 0;
  if (A.cut) len = min(len, max(A.cut[s], 0));
  return ok ? p : s;
}

__global__ __launch_bounds__(kThr) void fork_rows_kernel(ForkArgs A) {
  const Pages& st = A.st;
  const int s = blockIdx.x, mask = page_size(st) - 1;
  int len;
  const int p = fork_source(A, s, len);
  const int before = held(st, st.lens[s]);
  const int n = (len + mask) >> st.lg, m = (before + mask) >> st.lg;
  const int* from = st.table + static_cast<int64_t>(p) * st.width;
  const int* mine = st.table + static_cast<int64_t>(s) * st.width;
  int* to = A.rows + static_cast<int64_t>(s) * st.width;
  for (int j = threadIdx.x; j < max(n, m); j += kThr) {
    const int next = j < n ? page_id(st, from[j]) : -1;
    const int prev = j < m ? page_id(st, mine[j]) : -1;
    if (next != prev) {
      if (next >= 0) atomicAdd(&st.refs[next], 1);
      if (prev >= 0) atomicSub(&st.refs[prev], 1);
    }
    to[j] = next;
  }
  if (threadIdx.x == 0) A.lens[s] = len;
}

__global__ __launch_bounds__(kThr) void fork_place_kernel(ForkArgs A) {
  const Pages& st = A.st;
  const int s = blockIdx.x, mask = page_size(st) - 1;
  const int len = A.lens[s], before = held(st, st.lens[s]);
  const int n = (max(len, before) + mask) >> st.lg;
  for (int j = threadIdx.x; j < n; j += kThr)
    st.table[static_cast<int64_t>(s) * st.width + j] = A.rows[static_cast<int64_t>(s) * st.width + j];
  __syncthreads();  // (before is read by all)
  if (threadIdx.x == 0) {
    st.lens[s] = len;
    st.taken[s] = 0;
  }
}

struct CompactArgs {
  Pages st;
  int* moves;  // [1 + 2 * (pages / 2 + 1)]: their number, then where from ..
  int* to;     // .. and where to
  int* map;    // [pages]: where a page that moves goes
  int* in_use;
};

__global__ __launch_bounds__(kPlanThr) void compact_kernel(CompactArgs A) {
  __shared__ int s_wave[kPlanThr / 64];
  const Pages& st = A.st;
  const int tid = threadIdx.x;
  int n = 0;
  for (int base = 0; base < st.pages; base += 4 * kPlanThr) {
    int r[4], v = 0, sum;
    refs4(st, base + 4 * tid, 0, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) v += r[i] > 0 ? 1 : 0;
    block_prefix(v, s_wave, sum);
    n += sum;
  }
  // as many free pages lie below n as used ones do from n on
  int holes = 0, movers = 0;
  for (int base = 0; base < st.pages; base += 4 * kPlanThr) {
    const int p = base + 4 * tid;
    int r[4], v = 0, sum;
    refs4(st, p, 0, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p + i < n)
        v += r[i] <= 0 ? 1 : 0;
      else
        v += r[i] > 0 ? 1 << 16 : 0;
    }
    // (a strip of 4096 pages: both counts fit their 16 bits)
    const int at = block_prefix(v, s_wave, sum);
    int h = holes + (at & 0xffff), m = movers + (at >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p + i < n) {
        if (r[i] <= 0) A.to[h++] = p + i;
      } else if (r[i] > 0) {
        A.moves[1 + m++] = p + i;
      }
    }
    holes += sum & 0xffff;
    movers += sum >> 16;
  }
  __threadfence_block();
  __syncthreads();
  for (int i = tid; i < movers; i += kPlanThr) {
    const int from = A.moves[1 + i], to = A.to[i];
    A.map[from] = to;
    st.refs[to] = st.refs[from];
    st.refs[from] = 0;
  }
  if (tid == 0) {
    A.moves[0] = movers;
    A.in_use[0] = n;
  }
}

// Units: 1024 table entries each, then 16 KB of a page each.
__global__ __launch_bounds__(kThr) void move_kernel(CompactArgs A) {
  constexpr int kEntries = 1024, kPiece = 1024;  // (pieces of 16 bytes)
  const Pages& st = A.st;
  const int moves = A.moves[0], n = A.in_use[0];
  if (!moves) return;
  const int64_t entries = static_cast<int64_t>(st.seqs) * st.width, tables = (entries + kEntries - 1) / kEntries;
  const int64_t page = page_numbers(st) / 8;  // pieces
  const int64_t parts = (page + kPiece - 1) / kPiece, per = parts * st.layers;
  const int64_t units = tables + moves * per;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    if (u < tables) {
      for (int64_t i = u * kEntries + threadIdx.x; i < min((u + 1) * kEntries, entries); i += kThr) {
        const int p = st.table[i];
        if (p >= n && p < st.pages) st.table[i] = A.map[p];
      }
      continue;
    }
    const int64_t w = u - tables;
    const int64_t m = w / per, rest = w - m * per, layer = rest / parts, part = rest - layer * parts;
    u32x4* base = reinterpret_cast<u32x4*>(st.pool) + layer * st.pages * page;
    const u32x4* from = base + A.moves[1 + m] * page;
    u32x4* to = base + A.to[m] * page;
    const int64_t end = min((part + 1) * kPiece, page);
    for (int64_t i = part * kPiece + threadIdx.x; i < end; i += kThr) to[i] = from[i];
  }
}

struct RowsArgs {
  Pages st;
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_st, k_sh, v_st, v_sh;
  const int* cu;
  int64_t layer;
  int rows;
};

// Number of cu[0 .. S] that are at most row, by the lanes of a wave: one strip of 64 for up to 64 sequences.
__device__ __forceinline__ int entries_up_to(const int* cu, int S, int row) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = S + 1;  // the answer lies in lo .. lo + n
  while (n > 64) {
    const int step = (n + 63) / 64;
    const int i = lo + min((lane + 1) * step, n) - 1;  // the last entry of the lane's part
    const int full = __popcll(wave_ballot(cu[i] <= row));
    if (full == 64) return S + 1;
    n = min(step, n - full * step);
    lo += full * step;
    if (n <= 0) return lo;
  }
  return lo + __popcll(wave_ballot(lane < n && cu[lo + min(lane, n - 1)] <= row));
}

__global__ __launch_bounds__(kThr) void store_kernel(RowsArgs A) {
  const Pages& st = A.st;
  const int lane = threadIdx.x & 63;
  const int row = __builtin_amdgcn_readfirstlane(blockIdx.x * (kThr / 64) + (threadIdx.x >> 6));
  if (row >= A.rows) return;
  int s = row, i = 0;
  if (A.cu) {
    s = __builtin_amdgcn_readfirstlane(entries_up_to(A.cu, st.seqs, row)) - 1;
    if (s < 0 || s >= st.seqs) return;
    i = row - A.cu[s];
  }
  const int len = held(st, st.lens[s]), taken = st.taken[s];
  const int t = len - taken + i;
  if (i >= taken || t < 0) return;
  const int p = page_id(st, st.table[static_cast<int64_t>(s) * st.width + (t >> st.lg)]);
  const int64_t run = run_numbers(st);
  uint16_t* to = st.pool + (A.layer * st.pages + p) * page_numbers(st) + (t & (page_size(st) - 1)) * kD;
  const int pieces = st.H * (kD / 8);
  for (int e = lane; e < pieces; e += 64) {
    const int h = e >> 4, d = 8 * (e & 15);
    const u32x4 x = *reinterpret_cast<const u32x4*>(A.k + row * A.k_st + h * A.k_sh + d);
    const u32x4 y = *reinterpret_cast<const u32x4*>(A.v + row * A.v_st + h * A.v_sh + d);
    *reinterpret_cast<u32x4*>(to + h * run + d) = x;
    *reinterpret_cast<u32x4*>(to + (st.H + h) * run + d) = y;
  }
}

// A workgroup: 16 tokens of one (sequence, head), 16 pieces of 16 bytes each.
__global__ __launch_bounds__(kThr) void read_kernel(Pages st, int64_t layer, int n, uint16_t* k, uint16_t* v) {
  const int t = blockIdx.x * 16 + (threadIdx.x >> 4), d = 8 * (threadIdx.x & 15);
  const int h = blockIdx.y, s = blockIdx.z;
  if (t >= n) return;
  u32x4 x = u32x4{}, y = u32x4{};
  if (t < held(st, st.lens[s])) {
    const int p = page_id(st, st.table[static_cast<int64_t>(s) * st.width + (t >> st.lg)]);
    const int64_t run = run_numbers(st);
    const uint16_t* from =
        st.pool + (layer * st.pages + p) * page_numbers(st) + h * run + (t & (page_size(st) - 1)) * kD + d;
    x = *reinterpret_cast<const u32x4*>(from);
    y = *reinterpret_cast<const u32x4*>(from + st.H * run);
  }
  const int64_t at = ((static_cast<int64_t>(s) * st.H + h) * n + t) * kD + d;
  *reinterpret_cast<u32x4*>(k + at) = x;
  *reinterpret_cast<u32x4*>(v + at) = y;
}

// Workgroups of a launch that takes `units` pieces of work in turn.
unsigned grid_for(int64_t units, int per_cu) {
  const int64_t most = static_cast<int64_t>(device_cu_count()) * per_cu;
  return static_cast<unsigned>(units < 1 ? 1 : (units < most ? units : most));
}

}  // namespace

int check_pages(const lkv_pages* p, const char* what) {
  LKV_REQUIRE(p, "%s: null pointer", what);
  LKV_REQUIRE(p->dtype == LKV_DTYPE_F16 || p->dtype == LKV_DTYPE_BF16, "%s: dtype %d (float16 or bfloat16 pages)", what,
              p->dtype);
  LKV_REQUIRE(p->page_size >= 16 && p->page_size <= 256 && (p->page_size & (p->page_size - 1)) == 0,
              "%s: page_size=%lld must be a power of two from 16 to 256", what, (long long)p->page_size);
  LKV_REQUIRE(p->layers >= 1 && p->layers < (1 << 16) && p->pages >= 1 && p->pages < (1ll << 28) && p->kv_heads >= 1 &&
                  p->kv_heads < (1 << 15),
              "%s: layers=%lld pages=%lld kv_heads=%lld out of range", what, (long long)p->layers, (long long)p->pages,
              (long long)p->kv_heads);
  LKV_REQUIRE(p->seqs >= 1 && p->seqs <= kMaxSeqs, "%s: seqs=%lld must be 1 .. %d", what, (long long)p->seqs, kMaxSeqs);
  LKV_REQUIRE(p->width >= 1 && p->width * p->page_size < (1ll << 30), "%s: width=%lld out of range", what,
              (long long)p->width);
  // (extend counts the pages that all sequences ask for in 32 bits: a row of the table and a copy each at most, whatever cu holds)
  LKV_REQUIRE(p->seqs * (p->width + 1) < (1ll << 31), "%s: a table of %lld x %lld pages (2^31 are the most)", what,
              (long long)p->seqs, (long long)p->width);
  LKV_REQUIRE(p->pool && p->table && p->lens && p->refs && p->taken, "%s: null pointer", what);
  LKV_REQUIRE(aligned16(p->pool) && aligned4(p->table) && aligned4(p->lens) && aligned4(p->refs) && aligned4(p->taken),
              "%s: the pool must be 16-byte aligned, table, lens, refs and taken 4-byte", what);
  return LKV_OK;
}

Pages device_pages(const lkv_pages* p) {
  Pages st;
  st.pool = static_cast<uint16_t*>(p->pool);
  st.table = p->table;
  st.lens = p->lens;
  st.refs = p->refs;
  st.taken = p->taken;
  st.layers = static_cast<int>(p->layers);
  st.pages = static_cast<int>(p->pages);
  st.H = static_cast<int>(p->kv_heads);
  st.lg = 0;
  while ((1 << st.lg) < p->page_size) ++st.lg;
  st.seqs = static_cast<int>(p->seqs);
  st.width = static_cast<int>(p->width);
  return st;
}

int check_rows(const void* x, const int64_t* strides, const char* what, const char* name) {
  LKV_REQUIRE(x && strides, "%s: null pointer", what);
  LKV_REQUIRE(aligned16(x) && strides[0] >= 0 && strides[1] >= 0 && (strides[0] | strides[1]) % 8 == 0 &&
                  (strides[0] | strides[1]) < (1ll << 31),
              "%s: rows of %s must be 16-byte aligned, strides %lld, %lld", what, name, (long long)strides[0],
              (long long)strides[1]);
  return LKV_OK;
}

}  // namespace pages
}  // namespace lkv

using namespace lkv;
using namespace lkv::pages;

extern "C" size_t lkv_pages_extend_workspace_bytes(int64_t pages, int64_t seqs) {
  if (pages < 1 || seqs < 1) return 0;
  return static_cast<size_t>(pages + 1 + 3 * seqs) * 4;
}

extern "C" int lkv_pages_extend(const lkv_pages* p, const int32_t* cu, void* workspace, size_t workspace_bytes,
                                void* stream) {
  const char* what = "pages_extend";
  if (int rc = check_pages(p, what)) return rc;
  const size_t need = lkv_pages_extend_workspace_bytes(p->pages, p->seqs);
  LKV_REQUIRE(workspace && aligned4(workspace) && workspace_bytes >= need,
              "%s: a 4-byte aligned workspace of %zu bytes required, got %zu", what, need, workspace_bytes);
  LKV_REQUIRE(aligned4(cu), "%s: cu must be 4-byte aligned", what);
  const Pages st = device_pages(p);
  ExtendArgs A{st, cu, static_cast<int*>(workspace), static_cast<int*>(workspace) + p->pages};
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(extend_kernel, dim3(1), dim3(kPlanThr), 0, s, A);
  LKV_LAUNCH_CHECK("pages_extend");
  const dim3 grid(grid_for(p->seqs * p->layers * 2 * p->kv_heads, 4));
  hipLaunchKernelGGL(copy_kernel, grid, dim3(kThr), 0, s, st, A.copies);
  LKV_LAUNCH_CHECK("pages_extend copies");
  return LKV_OK;
}

extern "C" int lkv_pages_store(const lkv_pages* p, int64_t layer, const void* k, const int64_t* k_strides,
                               const void* v, const int64_t* v_strides, int64_t rows, const int32_t* cu, void* stream) {
  const char* what = "pages_store";
  if (int rc = check_pages(p, what)) return rc;
  LKV_REQUIRE(layer >= 0 && layer < p->layers, "%s: layer %lld of %lld", what, (long long)layer, (long long)p->layers);
  LKV_REQUIRE(rows >= 0 && rows < (1ll << 30), "%s: rows=%lld out of range", what, (long long)rows);
  LKV_REQUIRE(cu || rows == p->seqs || rows == 0, "%s: one row for each of %lld sequences, got %lld", what,
              (long long)p->seqs, (long long)rows);
  if (rows == 0) return LKV_OK;
  if (int rc = check_rows(k, k_strides, what, "k")) return rc;
  if (int rc = check_rows(v, v_strides, what, "v")) return rc;
  LKV_REQUIRE(aligned4(cu), "%s: cu must be 4-byte aligned", what);
  const RowsArgs A{device_pages(p), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), k_strides[0],
                   k_strides[1], v_strides[0], v_strides[1], cu, layer, static_cast<int>(rows)};
  const dim3 grid(static_cast<unsigned>((rows + kThr / 64 - 1) / (kThr / 64)));
  hipLaunchKernelGGL(store_kernel, grid, dim3(kThr), 0, static_cast<hipStream_t>(stream), A);
  LKV_LAUNCH_CHECK("pages_store");
  return LKV_OK;
}

extern "C" int lkv_pages_read(const lkv_pages* p, int64_t layer, int64_t n, void* k, void* v, void* stream) {
  const char* what = "pages_read";
  if (int rc = check_pages(p, what)) return rc;
  LKV_REQUIRE(layer >= 0 && layer < p->layers, "%s: layer %lld of %lld", what, (long long)layer, (long long)p->layers);
  LKV_REQUIRE(n >= 0 && n <= p->width * p->page_size, "%s: n=%lld outside sequences of up to %lld tokens", what,
              (long long)n, (long long)(p->width * p->page_size));
  if (n == 0) return LKV_OK;
  LKV_REQUIRE(k && v && aligned16(k) && aligned16(v), "%s: k and v must be 16-byte aligned", what);
  const dim3 grid(static_cast<unsigned>((n + 15) / 16), static_cast<unsigned>(p->kv_heads),
                  static_cast<unsigned>(p->seqs));
  hipLaunchKernelGGL(read_kernel, grid, dim3(kThr), 0, static_cast<hipStream_t>(stream), device_pages(p), layer,
                     static_cast<int>(n), static_cast<uint16_t*>(k), static_cast<uint16_t*>(v));
  LKV_LAUNCH_CHECK("pages_read");
  return LKV_OK;
}

extern "C" size_t lkv_pages_fork_workspace_bytes(int64_t seqs, int64_t width) {
  if (seqs < 1 || width < 1) return 0;
  return static_cast<size_t>(seqs * width + seqs) * 4;
}

extern "C" int lkv_pages_fork(const lkv_pages* p, const int32_t* parent, const int32_t* cut, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const char* what = "pages_fork";
  if (int rc = check_pages(p, what)) return rc;
  const size_t need = lkv_pages_fork_workspace_bytes(p->seqs, p->width);
  LKV_REQUIRE(workspace && aligned4(workspace) && workspace_bytes >= need,
              "%s: a 4-byte aligned workspace of %zu bytes required, got %zu", what, need, workspace_bytes);
  LKV_REQUIRE(aligned4(parent) && aligned4(cut), "%s: parent and cut must be 4-byte aligned", what);
  int* ws = static_cast<int*>(workspace);
  const ForkArgs A{device_pages(p), parent, cut, ws, ws + p->seqs * p->width};
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(fork_rows_kernel, dim3(static_cast<unsigned>(p->seqs)), dim3(kThr), 0, s, A);
  LKV_LAUNCH_CHECK("pages_fork");
  hipLaunchKernelGGL(fork_place_kernel, dim3(static_cast<unsigned>(p->seqs)), dim3(kThr), 0, s, A);
  LKV_LAUNCH_CHECK("pages_fork rows");
  return LKV_OK;
}

extern "C" size_t lkv_pages_compact_workspace_bytes(int64_t pages) {
  if (pages < 1) return 0;
  return static_cast<size_t>(1 + 2 * (pages / 2 + 1) + pages) * 4;
}

extern "C" int lkv_pages_compact(const lkv_pages* p, int32_t* in_use, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  const char* what = "pages_compact";
  if (int rc = check_pages(p, what)) return rc;
  const size_t need = lkv_pages_compact_workspace_bytes(p->pages);
  LKV_REQUIRE(workspace && aligned4(workspace) && workspace_bytes >= need,
              "%s: a 4-byte aligned workspace of %zu bytes required, got %zu", what, need, workspace_bytes);
  LKV_REQUIRE(in_use && aligned4(in_use), "%s: in_use must be 4-byte aligned", what);
  int* ws = static_cast<int*>(workspace);
  const int64_t half = p->pages / 2 + 1;
  const CompactArgs A{device_pages(p), ws, ws + 1 + half, ws + 1 + 2 * half, in_use};
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(kPlanThr), 0, s, A);
  LKV_LAUNCH_CHECK("pages_compact");
  const int64_t pieces = p->page_size * kD * 2 * p->kv_heads / 8 / 1024 + 1;
  const dim3 grid(grid_for(p->seqs * p->width / 1024 + 1 + half * p->layers * pieces, 8));
  hipLaunchKernelGGL(move_kernel, grid, dim3(kThr), 0, s, A);
  LKV_LAUNCH_CHECK("pages_compact moves");
  return LKV_OK;
}
