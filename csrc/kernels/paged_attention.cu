// Attention over a paged K/V cache for a batch whose requests share prefixes.
//
// Token t = cu_q[i] + j of request i (n_i tokens in this call, lens[i] keys of its own including them) sees the
// prefix of its group, keys [0, p), and its own keys [0, lens[i] - n_i + j]:
//   out[t, h] = sum_k softmax_k(scale q[t, h] . k) v_k          (h of nh; kv head h / (nh / nkv))
// A row that sees nothing is zero (lse -inf). One decode token, several scored tokens and a whole prompt are
// the same call.
//
// Work is cut by *segments*: one per group (all tokens of the group against the prefix, read once for them) and
// one per request (its tokens against its own pages). The rows of a segment and kv head are (token, head of the
// kv group) pairs, cut into row tiles (*entries*); an entry x kv head is an *item* of `tiles` key tiles. All
// items' key tiles form one line that the CTAs share in equal contiguous parts of `per` tiles, so one long
// sequence and many unlike ones fill the GPU alike (within a tile) and a CTA's part of an item (*piece*) has
// its own running maximum and sum; pieces are joined afterwards by their log-sum-exp. The line is laid out by
// one small kernel from the device lengths (no host copy, the grid never changes: fit for a CUDA graph) and
// serves every layer of the step. An item costs its key tiles plus a few units for its start and end (loading its
// queries, filling the pipeline, writing its rows), so that a CTA with many short items gets fewer tiles.
#include "common.cuh"
#include "spans.h"
#include <cuda.h>
#include <cudaTypedefs.h>
#include <atomic>
#include <mutex>
#include <type_traits>

namespace {

constexpr float LOG2E_F = 1.4426950408889634f;
constexpr float LN2_F = 0.6931471805599453f;

// Programmatic dependent launch: the next kernel of the stream may start (its own wait holds it where it needs this
// one's results); wait until the kernels before have completed and their writes are visible.
__device__ __forceinline__ void pdl_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ───────────────────────── plan ─────────────────────────
// Two kernels share the work. STREAM (mma.sync) takes segments of at most 16 rows a kv head, whose time is the
// K/V stream; WIDE (tcgen05) takes those with more, whose products count. Each has its own line of key tiles.
// Segments: groups first, then requests.
constexpr int PLAN_MAGIC = 0x50415432;
constexpr int STREAM = 0, WIDE = 1, WIDE_BIT = 1 << 30;
enum : int { H_MAGIC = 0, H_STATUS, H_B, H_G, H_T, H_N, H_NH, H_NKV, H_D, H_SHIFT, H_EMPTY,
             H_E = 12, H_W = 14, H_PER = 16, H_ROWS = 18, H_INTS = 32 };  // from H_E on: [STREAM, WIDE]
constexpr int PLAN_THREADS = 1024;

struct Entry {   // one row tile of a segment
  int cum;       // units (key tiles and starts) of all items before this entry's
  int seg;       // segment: a group's prefix below G (the same keys for every row), else a request (causal)
  int tok0;      // first token
  int ntok;      // tokens
  int keys;      // keys of the segment
  int vis;       // keys the first token sees
  int row;       // rows of all items before this entry's
  int tiles;     // key tiles of each of its nkv items
};
static_assert(sizeof(Entry) == 32, "entry record");

struct PlanArgs {
  const int *cu_q, *lens, *cu_group, *prefix_lens;
  int T, B, G, nh, nkv, d, shift;
  int max_own, max_prefix;  // keys that fit a table row
  int wide_rows;            // segments of more rows a kv head are WIDE
  int tpt[2], kt[2], ctas[2], max_entries[2], start[2];
};

// int32 buffer: header, each segment's first entry (WIDE_BIT: of that kernel; -1: none), each request's group, then
// the entry records of both kernels
__host__ __device__ inline int* plan_requests(int* plan, int segs) { return plan + H_INTS + (segs + 7) / 8 * 8; }
__host__ __device__ inline Entry* plan_entries(int* plan, int segs, int requests, int which, int max_stream) {
  return reinterpret_cast<Entry*>(plan_requests(plan, segs) + (requests + 7) / 8 * 8) + (which ? max_stream : 0);
}

struct Segment {
  int tok0, ntok, keys, vis, which;
};
__device__ __forceinline__ int tiles_of(int seen, int kt) { return (max(seen, 0) + kt - 1) / kt; }
__device__ __forceinline__ int units_of(int tiles, int start) { return tiles > 0 ? tiles + start : 0; }

// lane l's segment
__device__ __forceinline__ Segment segment_of(const Segment& g, int l) {
  return Segment{__shfl_sync(0xffffffffu, g.tok0, l), __shfl_sync(0xffffffffu, g.ntok, l), __shfl_sync(0xffffffffu, g.keys, l),
                 __shfl_sync(0xffffffffu, g.vis, l), __shfl_sync(0xffffffffu, g.which, l)};
}
constexpr int PLAN_ALONE = 4;  // row tiles that a segment's thread lays out itself; its warp does more together

// Sums of a chunk of segments that the scan carries: entries and key tiles of both kernels, rows of partial results.
struct Sums {
  long long entries;      // WIDE in the upper half, STREAM in the lower
  long long tiles[2], rows[2];  // (tiles with their items' start units)
  __device__ void add(const Sums& o) {
    entries += o.entries;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      tiles[w] += o.tiles[w];
      rows[w] += o.rows[w];
    }
  }
};
__device__ __forceinline__ Sums shifted_up(const Sums& v, int o) {
  Sums r;
  r.entries = __shfl_up_sync(0xffffffffu, v.entries, o);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    r.tiles[w] = __shfl_up_sync(0xffffffffu, v.tiles[w], o);
    r.rows[w] = __shfl_up_sync(0xffffffffu, v.rows[w], o);
  }
  return r;
}

// One block, a thread a segment (a warp for those of many row tiles): read its lengths, count its entries and key tiles,
// scan, write its entries. Bound: latency (two dependent reads, one scan: 3 to 4 us); a whole decode batch is one turn
// of the loop.
__global__ void __launch_bounds__(PLAN_THREADS) paged_plan_kernel(const PlanArgs a, int* __restrict__ plan) {
  __shared__ Sums s_warp[PLAN_THREADS / 32];
  __shared__ int s_empty;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5, S = a.G + a.B;
  int* seg_first = plan + H_INTS;
  int* request = plan_requests(plan, S);
  const int gsz = a.nh / a.nkv;
  pdl_next();
  if (tid == 0) s_empty = 0;
  Sums base{};  // of the chunks before this one
  int status = 0, empty = 0;
  for (int s0 = 0; s0 < S && !status; s0 += blockDim.x) {
    const int s = s0 + tid;
    Segment g{};
    bool bad = false;
    if (s < a.G) {
      const int g0 = a.cu_group[s], g1 = a.cu_group[s + 1], p = a.prefix_lens[s];
      bad = g0 < 0 || g1 < g0 || g1 > a.B || (s == 0 && g0 != 0) || (s == a.G - 1 && g1 != a.B) || p < 0 || p > a.max_prefix;
      if (!bad) {
        g.tok0 = a.cu_q[g0];
        g.ntok = a.cu_q[g1] - g.tok0;
        g.keys = g.vis = p;
        bad = g.tok0 < 0 || g.ntok < 0 || g.tok0 + g.ntok > a.T;
        if (!bad && a.G > 1)
          for (int i = g0; i < g1; ++i) request[i] = s;
      }
    } else if (s < S) {
      const int i = s - a.G, c0 = a.cu_q[i], c1 = a.cu_q[i + 1], n = a.lens[i];
      bad = c0 < 0 || c1 < c0 || c1 > a.T || (i == 0 && c0 != 0) || n < 0 || n > a.max_own;
      if (a.G == 1) request[i] = 0;
      if (!bad) {
        g.tok0 = c0;
        g.ntok = c1 - c0;
        g.keys = n;
        g.vis = n - g.ntok + 1;  // below 1 for tokens that see no key of their own
        empty += max(0, min(g.ntok, g.ntok - n));
      }
    }
    const bool causal = s >= a.G;
    g.which = (long long)g.ntok * gsz > a.wide_rows ? WIDE : STREAM;
    const int w = g.which, tpt = a.tpt[w], n = !bad && g.keys > 0 ? (g.ntok + tpt - 1) / tpt : 0;
    Sums v{};
    v.entries = w ? (long long)n << 32 : n;
    // units of row tile r of a segment
    auto units = [&](const Segment& f, bool own, int r) {
      const int t = a.tpt[f.which], seen = own ? min(f.keys, f.vis + min((r + 1) * t, f.ntok) - 1) : f.keys;
      return units_of(tiles_of(seen, a.kt[f.which]), a.start[f.which]);
    };
    long long sum = 0;
    for (int r = 0; r < (n <= PLAN_ALONE ? n : 0); ++r) sum += units(g, causal, r);
    for (unsigned todo = __ballot_sync(0xffffffffu, n > PLAN_ALONE); todo; todo &= todo - 1) {
      const int l = __ffs(todo) - 1, nl = __shfl_sync(0xffffffffu, n, l);
      const Segment f = segment_of(g, l);
      const bool own = __shfl_sync(0xffffffffu, (int)causal, l) != 0;
      long long part = 0;
      for (int r = lane; r < nl; r += 32) part += units(f, own, r);
#pragma unroll
      for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      if (lane == l) sum = part;
    }
    v.tiles[w] = sum * a.nkv;
    v.rows[w] = n ? (long long)g.ntok * a.nh : 0;
    Sums incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const Sums u = shifted_up(incl, o);
      if (lane >= o) incl.add(u);
    }
    if (lane == 31) s_warp[warp] = incl;
    if (__syncthreads_or(bad)) {
      status = 1;
      break;
    }
    if (warp == 0) {
      Sums t = lane < nw ? s_warp[lane] : Sums{};
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const Sums u = shifted_up(t, o);
        if (lane >= o) t.add(u);
      }
      if (lane < nw) s_warp[lane] = t;
    }
    __syncthreads();
    Sums at = base;
    if (warp) at.add(s_warp[warp - 1]);
    at.add(incl);  // through this segment; its own part comes off again below
    const int first = (int)((at.entries - v.entries) >> (w ? 32 : 0));
    base.add(s_warp[nw - 1]);
    // (the first cannot happen for lengths that passed; it keeps writes inside the buffer)
    if ((int)(base.entries & 0xffffffffLL) > a.max_entries[STREAM] || (int)(base.entries >> 32) > a.max_entries[WIDE])
      status = 2;
    else if (base.tiles[0] > 0x7fffffffLL - 4096 || base.tiles[1] > 0x7fffffffLL - 4096)
      status = 3;  // 2^31 key tiles in one call
    int cum = (int)(at.tiles[w] - v.tiles[w]), row = (int)(at.rows[w] - v.rows[w]);
    auto write = [&](const Segment& f, bool own, int seg, int to, int r, int at_unit, int at_row) {
      const int t = a.tpt[f.which], j0 = r * t;
      Entry e;
      e.cum = at_unit;
      e.seg = seg;
      e.tok0 = f.tok0 + j0;
      e.ntok = min(t, f.ntok - j0);
      e.keys = f.keys;
      e.vis = f.vis + (own ? j0 : 0);
      e.row = at_row + j0 * a.nh;
      e.tiles = tiles_of(min(f.keys, e.vis + (own ? e.ntok - 1 : 0)), a.kt[f.which]);
      plan_entries(plan, S, a.B, f.which, a.max_entries[STREAM])[to + r] = e;
    };
    if (s < S && !status) {
      seg_first[s] = n ? first | (w ? WIDE_BIT : 0) : -1;
      for (int r = 0; r < (n <= PLAN_ALONE ? n : 0); ++r) {
        write(g, causal, s, first, r, cum, row);
        cum += units(g, causal, r) * a.nkv;
      }
    }
    for (unsigned todo = __ballot_sync(0xffffffffu, n > PLAN_ALONE && !status); todo; todo &= todo - 1) {
      const int l = __ffs(todo) - 1, nl = __shfl_sync(0xffffffffu, n, l), to = __shfl_sync(0xffffffffu, first, l);
      const Segment f = segment_of(g, l);
      const bool own = __shfl_sync(0xffffffffu, (int)causal, l) != 0;
      int c = __shfl_sync(0xffffffffu, cum, l);
      const int rw = __shfl_sync(0xffffffffu, row, l);
      for (int r0 = 0; r0 < nl; r0 += 32) {
        const int r = r0 + lane, mine = r < nl ? units(f, own, r) * a.nkv : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += u;
        }
        if (r < nl) write(f, own, s - lane + l, to, r, c + upto - mine, rw);
        c += __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    __syncthreads();  // s_warp is free again
  }
  if (empty) atomicAdd(&s_empty, empty);
  __syncthreads();
  if (tid == 0) {
    if (status) dt_report(DT_ERR_BAD_ARG, 710 + status);
    plan[H_MAGIC] = PLAN_MAGIC;
    plan[H_STATUS] = status;
    plan[H_B] = a.B;
    plan[H_G] = a.G;
    plan[H_T] = a.T;
    plan[H_N] = status ? 0 : a.cu_q[a.B];
    plan[H_NH] = a.nh;
    plan[H_NKV] = a.nkv;
    plan[H_D] = a.d;
    plan[H_SHIFT] = a.shift;
    plan[H_EMPTY] = s_empty;
    for (int w = 0; w < 2; ++w) {
      const long long W = status ? 0 : base.tiles[w];
      plan[H_E + w] = status ? 0 : (int)(w ? base.entries >> 32 : base.entries & 0xffffffffLL);
      plan[H_W + w] = (int)W;
      plan[H_PER + w] = W ? (int)((W + a.ctas[w] - 1) / a.ctas[w]) : 1;
      plan[H_ROWS + w] = status ? 0 : (int)base.rows[w];
    }
  }
}

// ───────────────────────── shared by the kernels below ─────────────────────────
struct AttnArgs {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  float* lse;        // [T, nh] or null
  const int* plan;
  const int *tables, *prefix_tables;
  long long ld_tables, ld_prefix;
  const int *cu_q, *cu_group;
  float* part_o;     // [row][D] partial results
  float* part_lse;   // [row], log2
  int T, B, G, nh, nkv, shift, pages, max_stream;
  int stream_ctas;
  // The order of the two kernels. The first waits for what is in front of it; the second starts once every block of the
  // first has passed that wait, so the plan and all before it are there, while the first may still run: each block of
  // the second waits for it before it ends, for the join behind both.
  int wide_first;
  int start[2];      // start units of an item
  float scale;
};
constexpr int STREAM_ROWS = 16, WIDE_ROWS = 256;

// The plan is read through L2: a kernel that starts early (see pdl_wait) must not meet lines of the last step's plan.
__device__ __forceinline__ Entry load_entry(const Entry* p) {
  const int4* q = reinterpret_cast<const int4*>(p);
  const int4 a = __ldcg(q), b = __ldcg(q + 1);
  return Entry{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}

// the entry that holds key tile x: last e with cum <= x (entries without tiles share their successor's cum).
// 32 probes a round, so a few hundred entries take two round trips.
__device__ __forceinline__ int find_entry(const Entry* ent, int E, int x, int lane) {
  int lo = 0, hi = E;  // answer in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + lane * step;
    const bool le = at < hi && __ldcg(&ent[at].cum) <= x;
    const unsigned m = __ballot_sync(0xffffffffu, le);
    const int last = 31 - __clz(m);  // lane 0 always holds (cum of lo <= x)
    const int nlo = lo + last * step;
    hi = min(hi, nlo + step);
    lo = nlo;
  }
  return lo;
}

// Whether dynamic shared memory starts off a 1024-byte border, which the swizzles rely on (it does once a kernel has
// static shared memory too, whatever alignment the array is declared with; the test must not be folded by that).
__device__ __forceinline__ bool misaligned(const void* smem) {
  uint32_t a = smem_u32(smem);
  asm volatile("" : "+r"(a));
  return (a & 1023u) != 0;
}

// The plan's header for a whole block: one thread reads it (thousands of warps asking L2 for the same line would
// wait for each other), and says whether it is this call's.
struct Header {
  int v[H_INTS];
  __device__ int operator[](int i) const { return v[i]; }
  __device__ bool load(const AttnArgs& a, int D) {  // every thread of the block calls this
    if (threadIdx.x < H_INTS) v[threadIdx.x] = __ldcg(a.plan + threadIdx.x);
    __syncthreads();
    return v[H_MAGIC] == PLAN_MAGIC && v[H_B] == a.B && v[H_G] == a.G && v[H_T] == a.T && v[H_NH] == a.nh &&
           v[H_NKV] == a.nkv && v[H_D] == D && v[H_SHIFT] == a.shift;
  }
};

// A CTA's part of an item: key tiles t0 .. t1 of the item (kv head h), from line position x up to `next`. Parts that
// hold start units alone have no tiles.
struct Piece {
  int h, t0, t1, next;
};
__device__ __forceinline__ Piece piece_at(const Entry& en, int x, int x1, int start) {
  const int units = en.tiles + start, loc = x - en.cum;
  Piece p;
  p.h = loc / units;
  const int u0 = loc - p.h * units, u1 = min(units, u0 + (x1 - x));
  p.t0 = max(u0 - start, 0);
  p.t1 = max(u1 - start, 0);
  p.next = x + (u1 - u0);
  return p;
}

// First row of a piece's partial result. With groups every piece is kept: an item's rows follow those of the
// items before it, and each CTA shifts them by a whole tile more, so two pieces of one item do not meet.
// Without, only the two pieces at the ends of a CTA's part can be incomplete.
__device__ __forceinline__ long long piece_row(const AttnArgs& a, const Header& head, int which, const Entry& en,
                                               int h, int cta, int first, int per) {
  const int tile = which ? WIDE_ROWS : STREAM_ROWS;
  if (a.G == 0) {
    const long long base = which ? 2LL * a.stream_ctas * STREAM_ROWS : 0;
    return base + (2LL * cta + (first != cta * per ? 1 : 0)) * tile;
  }
  const long long base = which ? (long long)head[H_ROWS + STREAM] + (long long)a.stream_ctas * STREAM_ROWS : 0;
  return base + en.row + (long long)h * en.ntok * (a.nh / a.nkv) + (long long)cta * tile;
}

// ───────────────────────── STREAM: mma.sync ─────────────────────────
// At most 16 rows an item (a decode token's kv group; head dims below 64 take several entries for more). Bound: HBM
// - 2 * 16 * d flops a key against 4 d bytes - so the kernel is a stream. One producer warp walks the line: for each
// piece it leaves a descriptor and its queries in one of two slots, then keeps TMA loads of K and V in flight
// through a ring of stages, running ahead of the consumers across pieces (it looks the next entry and its page ids
// up while the current piece loads). Four warps take whole stages in turn (S = Q K^T, online softmax, O += P V in
// registers, each warp with its own maximum and sum) and meet only at the end of a piece. Two CTAs an SM.
// Page boxes land in the swizzle of their row width (128 / 64 / 32 bytes), so ldmatrix reads do not conflict.
// Rows of V past the segment's last key (the rest of its last page may hold anything) are zeroed in shared
// memory before use, masked scores are replaced, never added to: what lies there cannot reach a result.
// Measured: 55 us for the decode step of 64 requests of up to 4095 keys, 16 heads on 4, d = 128 (328 MB: 6.0 TB/s, 0.91
// of a plain copy's rate); 36 us for the own keys of 128 answers over a shared prompt (175 MB).
constexpr int DEC_WARPS = 4, DEC_THREADS = 32 * (1 + DEC_WARPS), DEC_ROWS = STREAM_ROWS, DEC_CTAS = 2;

template <int D>
struct DCfg {
  static constexpr int KT = D == 128 ? 32 : 64;                // keys a tile
  static constexpr int CW = D < 64 ? D : 64;                   // columns of a box
  static constexpr int RB = CW * 2;                            // bytes of a box row = swizzle width
  static constexpr int HALF = KT * D * 2;                      // K (or V) bytes of a stage
  static constexpr int MC = D < 64 ? D : 64;                   // columns joined at a time
  static constexpr int MERGE = DEC_WARPS * DEC_ROWS * MC * 4;
  static constexpr int QB = DEC_ROWS * D * 2;                  // queries of a slot
  static constexpr int ST = D >= 64 ? 5 : 8;
  static constexpr int SMEM = ST * 2 * HALF + 2 * QB + MERGE + 2 * DEC_WARPS * DEC_ROWS * 4 + (2 * ST + 6) * 8 +
                              2 * 64 + 16 + 4 * H_INTS;
  static_assert(DEC_CTAS * (SMEM + 1024) <= 233472, "decode shared memory");
  static_assert(ST >= DEC_WARPS, "a warp's tiles wait on stages of its previous tile's time");
  // byte offset of 16-byte chunk c (of D / 8) of key row r inside a K or V stage
  __device__ static int at(int r, int c) {
    const int x = RB == 128 ? (r & 7) : RB == 64 ? ((r >> 1) & 3) : ((r >> 2) & 1);
    return (c / (CW / 8)) * (KT * RB) + r * RB + (((c % (CW / 8)) ^ x) << 4);
  }
  __device__ static int q_at(int r, int c) {  // the same inside a slot's queries
    const int x = RB == 128 ? (r & 7) : RB == 64 ? ((r >> 1) & 3) : ((r >> 2) & 1);
    return (c / (CW / 8)) * (DEC_ROWS * RB) + r * RB + (((c % (CW / 8)) ^ x) << 4);
  }
};

// What the consumers need to know of a piece (tiles = 0: there are no more).
struct StreamPiece {
  int tiles, key0, keys, vis, causal, rows, tok0, head0, direct, pad;
  long long part;
};
static_assert(sizeof(StreamPiece) <= 64, "descriptor slot");

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Bounded wait of a whole warp: every lane polls and the outcome is a vote, so the warp stays converged. (With one
// lane polling and the others waiting for its word the products behind the wait were issued from a warp that had
// not come together again: 270 clocks an MMA instead of 30.) Gives up like mbar_wait_bounded.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int err, int site, volatile int* abort_flag,
                                          int lane) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const uint64_t t0 = dt_globaltimer();
  uint32_t it = 0;
  while (true) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((++it & 255u) == 0) {
      const bool late = dt_globaltimer() - t0 > DT_WAIT_NS;
      if (__any_sync(0xffffffffu, late || *abort_flag || *reinterpret_cast<volatile int*>(&dt_error_word) != 0)) {
        if (lane == 0) {
          if (late) dt_set_error(err, site);
          *abort_flag = 1;
        }
        __syncwarp();
        return false;
      }
    }
  }
}

template <int D>
__global__ void __launch_bounds__(DEC_THREADS, DEC_CTAS)
paged_stream_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const AttnArgs a) {
  using C = DCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem;                                                     // [ST][K | V]
  uint8_t* sQ = ring + C::ST * 2 * C::HALF;                                 // [2][QB]
  float* mergeO = reinterpret_cast<float*>(sQ + 2 * C::QB);                 // [warp][16][MC]
  float* mergeM = mergeO + DEC_WARPS * DEC_ROWS * C::MC;                    // [warp][16]
  float* mergeL = mergeM + DEC_WARPS * DEC_ROWS;
  StreamPiece* piece = reinterpret_cast<StreamPiece*>(mergeL + DEC_WARPS * DEC_ROWS);  // [2], 64 bytes apart
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(piece) + 2 * 64);
  uint64_t* empty = full + C::ST;
  uint64_t* piece_full = empty + C::ST;   // [2]
  uint64_t* piece_empty = piece_full + 2; // [2]
  uint64_t* meet = piece_empty + 2;       // [2] the consumers' meeting points, in turn
  volatile int* abort_flag = reinterpret_cast<volatile int*>(meet + 2);
  Header& head = *reinterpret_cast<Header*>(const_cast<int*>(abort_flag) + 2);
  auto slot = [&](int i) -> StreamPiece& { return *reinterpret_cast<StreamPiece*>(reinterpret_cast<uint8_t*>(piece) + 64 * (i & 1)); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (misaligned(smem)) {  // uniform across the CTA
    if (threadIdx.x == 0) dt_set_error(DT_ERR_BAD_ARG, 720);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&piece_full[i], 1);
      mbar_init(&piece_empty[i], DEC_WARPS);
      mbar_init(&meet[i], DEC_WARPS);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (!a.wide_first) pdl_wait();  // the plan, and the cache and queries that the kernels before it wrote (see AttnArgs)
  pdl_next();
  if (!head.load(a, D)) {
    if (threadIdx.x == 0 && blockIdx.x == 0) dt_report(DT_ERR_BAD_ARG, 721);
    pdl_wait();
    return;
  }
  const int W = head[H_W + STREAM], per = head[H_PER + STREAM], E = head[H_E + STREAM];
  const Entry* ent = plan_entries(const_cast<int*>(a.plan), a.G + a.B, a.B, STREAM, a.max_stream);
  const long long x0l = (long long)blockIdx.x * per;
  if (x0l >= W) {
    pdl_wait();
    return;
  }
  const int x0 = (int)x0l, x1 = min(W, x0 + per);
  const int gsz = a.nh / a.nkv;
  const int P = 1 << a.shift;

  if (warp == 0) {
    // ───── producer ─────
    const int box_rows = min(P, C::KT), boxes = C::KT / box_rows;
    const int none = a.pages * a.nkv * P;  // a row past the cache: the box is filled with zeros
    const int tpt = DEC_ROWS / gsz;
    int e = find_entry(ent, E, x0, lane);
    Entry en = load_entry(ent + e);
    auto table_of = [&](const Entry& f) {
      return f.seg < a.G ? a.prefix_tables + f.seg * a.ld_prefix : a.tables + (f.seg - a.G) * a.ld_tables;
    };
    // 32 page ids of an entry's table from page p on, one a lane (-1: outside the cache)
    auto window = [&](const Entry& f, int p) {
      p += lane;
      int id = p * P < f.keys ? __ldcg(table_of(f) + p) : 0;
      if (p * P < f.keys && (unsigned)id >= (unsigned)a.pages) {
        dt_report(DT_ERR_BOUNDS, 723);
        id = -1;
      }
      return id;
    };
    int jl = 0, pc = 0;
    bool ok = true;
    int ahead = -1, ahead_win = 0;  // first page ids of the next piece, already requested (ahead: its first page)
    for (int x = x0; x < x1 && ok;) {
      const Piece pi = piece_at(en, x, x1, a.start[STREAM]);
      // the entry of the piece after this one
      const bool more = pi.next < x1;
      const bool same = pi.next < en.cum + (en.tiles + a.start[STREAM]) * a.nkv;
      int e2 = e;
      if (more && !same) {
        ++e2;
        while (e2 + 1 < E && __ldcg(&ent[e2].tiles) == 0) ++e2;
      }
      Entry en2 = more && !same ? load_entry(ent + e2) : en;
      if (pi.t1 > pi.t0) {
        if (pc >= 2) ok = warp_wait(&piece_empty[pc & 1], ((pc >> 1) & 1) ^ 1, DT_ERR_TIMEOUT_EMPTY, 726, abort_flag, lane);
        if (!ok) break;
        if (lane == 0) {
          StreamPiece d;
          d.tiles = pi.t1 - pi.t0;
          d.key0 = pi.t0 * C::KT;
          d.keys = en.keys;
          d.vis = en.vis;
          d.causal = en.seg >= a.G;
          d.rows = en.ntok * gsz;
          d.tok0 = en.tok0;
          d.head0 = pi.h * gsz;
          d.direct = a.G == 0 && pi.t0 == 0 && pi.t1 == en.tiles;
          d.pad = 0;
          d.part = piece_row(a, head, STREAM, en, pi.h, blockIdx.x, x, per);
          slot(pc) = d;
          mbar_arrive_expect_tx(&piece_full[pc & 1], tpt * gsz * C::RB * (D / C::CW));
#pragma unroll
          for (int c = 0; c < D / C::CW; ++c)
            tma_load_3d(sQ + (pc & 1) * C::QB + c * DEC_ROWS * C::RB, &tmQ, &piece_full[pc & 1], c * C::CW, pi.h * gsz,
                        en.tok0);
        }
        __syncwarp();
        ++pc;
        int win0 = (pi.t0 * C::KT) >> a.shift;
        int win = ahead == win0 ? ahead_win : window(en, win0);
        ahead = -1;
        for (int t = pi.t0; t < pi.t1; ++t, ++jl) {
          const int st = jl % C::ST;
          if (jl >= C::ST) ok = warp_wait(&empty[st], ((jl / C::ST) & 1) ^ 1, DT_ERR_TIMEOUT_EMPTY, 722, abort_flag, lane);
          if (!ok) break;
          const int k0 = t * C::KT;
          const int p0 = k0 >> a.shift, p1 = (min(k0 + C::KT, en.keys) - 1) >> a.shift;
          if (p1 >= win0 + 32) {
            win0 = p0;
            win = window(en, p0);
          }
          if (lane == 0) mbar_arrive_expect_tx(&full[st], 2 * C::HALF);
          __syncwarp();
          // lane b fetches box b of K and V
          const int key = k0 + lane * box_rows;
          const int page = __shfl_sync(0xffffffffu, win, ((key >> a.shift) - win0) & 31);
          if (lane < boxes) {
            const int row = key < en.keys && page >= 0 ? (page * a.nkv + pi.h) * P + (key & (P - 1)) : none;
            uint8_t* dst = ring + st * 2 * C::HALF + lane * box_rows * C::RB;
#pragma unroll
            for (int c = 0; c < D / C::CW; ++c) {
              tma_load_2d(dst + c * C::KT * C::RB, &tmK, &full[st], c * C::CW, row);
              tma_load_2d(dst + C::HALF + c * C::KT * C::RB, &tmV, &full[st], c * C::CW, row);
            }
          }
          __syncwarp();
          // (once the ring has been filled: a look at the next piece must not hold up its own first loads)
          if (more && ahead < 0 && (t + 1 == pi.t1 || t - pi.t0 + 1 >= C::ST)) {
            ahead = 0;  // the next piece starts its item, at page 0
            ahead_win = window(en2, 0);
          }
        }
      }
      x = pi.next;
      e = e2;
      en = en2;
    }
    if (ok && pc >= 2) ok = warp_wait(&piece_empty[pc & 1], ((pc >> 1) & 1) ^ 1, DT_ERR_TIMEOUT_EMPTY, 727, abort_flag, lane);
    if (ok && lane == 0) {
      slot(pc).tiles = 0;
      mbar_arrive(&piece_full[pc & 1]);
    }
    // nothing may be in flight into shared memory when the CTA ends, not after an aborted run either (bounded)
    if (lane == 0) {
      const uint64_t w0 = dt_globaltimer();
      for (int k = max(0, jl - C::ST); k < jl; ++k)
        while (!mbar_try_wait(&full[k % C::ST], (k / C::ST) & 1) && dt_globaltimer() - w0 < 20000000ull) {}
      for (int k = max(0, pc - (ok ? 1 : 2)); k < pc; ++k)  // (the end mark went through the older slot)
        while (!mbar_try_wait(&piece_full[k & 1], (k >> 1) & 1) && dt_globaltimer() - w0 < 20000000ull) {}
    }
    pdl_wait();
    return;
  }

  // ───── consumers ─────
  const int cw = warp - 1, tid = threadIdx.x - 32;
  const float sl2 = a.scale * LOG2E_F;
  const int r0 = lane >> 2, c2 = (lane & 3) * 2;
  int jl = 0, met = 0;
  // all four warps reach this point (bounded, so a warp that gives up strands nobody)
  auto meet_all = [&](int site) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&meet[met & 1]);
    const bool ok = warp_wait(&meet[met & 1], (met >> 1) & 1, DT_ERR_TIMEOUT_FULL, site, abort_flag, lane);
    ++met;
    return ok;
  };
  for (int pc = 0;; ++pc) {
    if (!warp_wait(&piece_full[pc & 1], (pc >> 1) & 1, DT_ERR_TIMEOUT_FULL, 728, abort_flag, lane)) break;
    const StreamPiece d = slot(pc);
    if (d.tiles == 0) break;
    uint32_t qf[D / 16][4];
    {
      const uint32_t qu = smem_u32(sQ + (pc & 1) * C::QB);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) ldsm4(qf[k], qu + C::q_at(((lane >> 3) & 1) * 8 + (lane & 7), k * 2 + (lane >> 4)));
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&piece_empty[pc & 1]);
    int vis[2];  // keys rows r0 and r0 + 8 see; rows behind the last are computed like others and left out
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = r0 + 8 * u;
      vis[u] = r < d.rows && d.causal ? min(d.vis + r / gsz, d.keys) : d.keys;
    }
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    bool ok = true;
    for (int t = (cw - jl) & (DEC_WARPS - 1); t < d.tiles; t += DEC_WARPS) {  // tiles jl + t = cw (mod 4)
      const int j = jl + t, st = j % C::ST;
      // A stage's uses alternate between the warps, so this warp may be here before the stage's previous use has
      // even arrived, and a parity test alone would then pass on the phase before that. First wait for the
      // previous use's release: its own last tile (j - 4) was issued after use - 2 had been released (ST >= 4),
      // so that test cannot be off by a phase either.
      ok = (j < C::ST || warp_wait(&empty[st], ((j / C::ST) & 1) ^ 1, DT_ERR_TIMEOUT_EMPTY, 725, abort_flag, lane)) &&
           warp_wait(&full[st], (j / C::ST) & 1, DT_ERR_TIMEOUT_FULL, 724, abort_flag, lane);
      if (!ok) break;
      uint8_t* sk = ring + st * 2 * C::HALF;
      const uint32_t ku = smem_u32(sk), vu = ku + C::HALF;
      const int k0 = d.key0 + t * C::KT, valid = d.keys - k0;
      if (valid < C::KT) {  // the segment's last tile
        for (int i = lane; i < (C::KT - valid) * (D / 8); i += 32)
          *reinterpret_cast<uint4*>(sk + C::HALF + C::at(valid + i / (D / 8), i % (D / 8))) = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
      float s[C::KT / 8][4];
#pragma unroll
      for (int n = 0; n < C::KT / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
#pragma unroll
        for (int n = 0; n < C::KT / 8; n += 2) {  // 16 keys x 16 dims a load
          uint32_t b[4];
          ldsm4(b, ku + C::at((n + (lane >> 4)) * 8 + (lane & 7), k * 2 + ((lane >> 3) & 1)));
          mma_bf16(s[n], qf[k], b[0], b[1]);
          mma_bf16(s[n + 1], qf[k], b[2], b[3]);
        }
      }
      float mx[2] = {-INFINITY, -INFINITY};
      const bool whole = k0 + C::KT <= min(vis[0], vis[1]);
#pragma unroll
      for (int n = 0; n < C::KT / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[n][i] *= sl2;
          if (!whole && k0 + n * 8 + c2 + (i & 1) >= vis[i >> 1]) s[n][i] = -INFINITY;
          mx[i >> 1] = fmaxf(mx[i >> 1], s[n][i]);
        }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 1));
        mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 2));
        mx[u] = fmaxf(mx[u], m[u]);
      }
      const float ms[2] = {mx[0] == -INFINITY ? 0.f : mx[0], mx[1] == -INFINITY ? 0.f : mx[1]};
      const float al[2] = {ex2_approx(m[0] - ms[0]), ex2_approx(m[1] - ms[1])};
      m[0] = mx[0];
      m[1] = mx[1];
      l[0] *= al[0];
      l[1] *= al[1];
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        o[n][0] *= al[0];
        o[n][1] *= al[0];
        o[n][2] *= al[1];
        o[n][3] *= al[1];
      }
      // P in bf16 (an MMA operand); the sum takes the rounded values, so the weights add up to one
#pragma unroll
      for (int kk = 0; kk < C::KT / 16; ++kk) {
        uint32_t p[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int n = 2 * kk + (v >> 1), u = v & 1;
          p[v] = pack_bf16(ex2_approx(s[n][2 * u] - ms[u]), ex2_approx(s[n][2 * u + 1] - ms[u]));
          const float2 f = unpack_bf16(p[v]);
          l[u] += f.x + f.y;
        }
#pragma unroll
        for (int n = 0; n < D / 8; n += 2) {
          uint32_t b[4];
          ldsm4_t(b, vu + C::at(kk * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), n + (lane >> 4)));
          mma_bf16(o[n], p, b[0], b[1]);
          mma_bf16(o[n + 1], p, b[2], b[3]);
        }
      }
      if (valid < C::KT) fence_proxy_async_smem();  // zeroed rows (generic writes) before the stage's next TMA write
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
    if (!ok) break;
    jl += d.tiles;
    // ── join the four warps, 64 columns at a time ──
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
      l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
      if ((lane & 3) == 0) {
        mergeM[cw * DEC_ROWS + r0 + 8 * u] = m[u];
        mergeL[cw * DEC_ROWS + r0 + 8 * u] = l[u];
      }
    }
#pragma unroll
    for (int part = 0; part < D / C::MC; ++part) {
#pragma unroll
      for (int n = 0; n < C::MC / 8; ++n) {
        float* w = mergeO + (cw * DEC_ROWS + r0) * C::MC + n * 8 + c2;
        const float(&v)[4] = o[part * (C::MC / 8) + n];
        if (r0 < d.rows) *reinterpret_cast<float2*>(w) = make_float2(v[0], v[1]);
        if (r0 + 8 < d.rows) *reinterpret_cast<float2*>(w + 8 * C::MC) = make_float2(v[2], v[3]);
      }
      ok = meet_all(729);
      if (!ok) break;
      for (int i = tid; i < d.rows * (C::MC / 4); i += 32 * DEC_WARPS) {
        const int r = i / (C::MC / 4), c = i % (C::MC / 4) * 4;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < DEC_WARPS; ++w) mm = fmaxf(mm, mergeM[w * DEC_ROWS + r]);
        if (mm == -INFINITY) mm = 0.f;  // nothing seen (or only NaN): sums of zeros (or NaN)
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < DEC_WARPS; ++w) {
          const float f = ex2_approx(mergeM[w * DEC_ROWS + r] - mm);
          const float4 v = *reinterpret_cast<const float4*>(mergeO + (w * DEC_ROWS + r) * C::MC + c);
          sum += f * mergeL[w * DEC_ROWS + r];
          acc.x += f * v.x;
          acc.y += f * v.y;
          acc.z += f * v.z;
          acc.w += f * v.w;
        }
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        const float ls = sum != 0.f ? mm + log2f(sum) : -INFINITY;
        const int col = part * C::MC + c;
        if (d.direct) {
          const int tok = r / gsz;
          const long long row = (long long)(d.tok0 + tok) * a.nh + d.head0 + (r - tok * gsz);
          *reinterpret_cast<uint2*>(a.out + row * D + col) = make_uint2(pack_bf16(acc.x, acc.y), pack_bf16(acc.z, acc.w));
          if (a.lse && col == 0) a.lse[row] = ls * LN2_F;
        } else {
          *reinterpret_cast<float4*>(a.part_o + (d.part + r) * D + col) = acc;
          if (col == 0) a.part_lse[d.part + r] = ls;
        }
      }
      ok = meet_all(730);  // the buffers are read before they are written again
      if (!ok) break;
    }
    if (!ok) break;
  }
  pdl_wait();
}

// ───────────────────────── WIDE: tcgen05 ─────────────────────────
// An item is two tiles of up to 128 rows (whole tokens: 128 / group rows each) of one segment and kv head, over
// the same key tiles of 64. TMEM holds two score buffers of 64 columns and the output of each row tile (2 x 128 +
// 2 d columns; the weights P take the first half of the scores they come from). Each row tile has an MMA warp, which
// runs two key tiles ahead of the weights - S(0) S(1) | P(0): PV(0) S(2) | P(1): PV(1) S(3) | ... - so a softmax
// warp finds its next scores ready when it has handed over its weights.
//   warp 0      producer: a piece's record and Q of both tiles (3-D map [token][head][d], whole kv groups) into one of
//               two slots, so the next piece is there before the last is done, then K and V tiles through one ring
//               in the order of their use
//   warps 1-2   products of row tile 0 and 1. (One warp for both took 2100 clocks a pair of key tiles, most of it
//               the latency of its own waits; two take 1700.)
//   warps 4-11  softmax, one thread a row (warps 4-7 tile 0, 8-11 tile 1). The running maximum only moves when it
//               grows by more than 8 (log2): O is rescaled then, once the product before has completed, else P is
//               taken against the old one (<= 2^8)
// The segment's last V tile has its rows behind the last key zeroed (they may hold anything) by each row tile's
// softmax warps before they hand over P.
// Measured: a prompt's second part (4095 tokens behind 2048, 40 heads on 8, d = 128: 344 GFLOP) takes 310 us here, 1.1
// PFLOP/s of visible scores; tensor pipe and exponential unit are each busy 61% of the time. A pair of key tiles takes
// 1700 clocks: S of 64 columns reads Q again for each tile from shared memory (about 64 clocks an MMA instead of 32),
// so the products alone come to 1650; half of Q in TMEM as the A operand would save 5%, S of 128 columns has no room
// for two buffers and waits for its weights (376 us for the call with the row tiles taking turns, 402 without). A piece
// costs 4700 clocks more, mostly its output rows.
constexpr int BKV = 64;
constexpr int WIDE_THREADS = 128 + 256;
constexpr float RESCALE_THRESHOLD = 8.0f;

// A piece as the producer hands it to the other warps, with its Q.
struct alignas(16) WidePiece {
  int tiles;  // 0: the CTA's part is done
  int key0, keys, vis, causal, tok0, ntok, head0, direct, pad;
  long long part;
};
static_assert(sizeof(WidePiece) == 48, "piece record");

template <int D>
struct WCfg {
  static constexpr int TQ = 128 * D * 2;               // one [128][D] bf16 query tile in 64-column chunks
  static constexpr int TT = BKV * D * 2;               // one [64][D] K or V tile
  static constexpr int ST = D == 128 ? 6 : 12;         // ring stages
  static constexpr int SMEM = 4 * TQ + ST * TT + 2 * (int)sizeof(WidePiece) + (2 * ST + 16) * 8 + 16 + 4 * H_INTS;
  static constexpr int C_S = 0, C_O = 256, TMEM_COLS = 512;
  static_assert(SMEM <= 232448, "shared memory");
};

// Descriptor offsets (16-byte units) of the k-th 16 of the inner dimension: of a query tile, of a K tile, of a V tile.
__host__ __device__ constexpr uint64_t qoff(int k) { return (uint64_t)(((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4); }
__host__ __device__ constexpr uint64_t koff(int k) { return (uint64_t)(((k >> 2) * (BKV * 128) + (k & 3) * 32) >> 4); }
__host__ __device__ constexpr uint64_t voff(int k) { return (uint64_t)((k * 2048) >> 4); }

// Products and commits issued from a converged warp, one elected lane executing the instruction: the operands are
// warp-uniform values to the compiler (26 clocks of issue an MMA; about 130 from inside a one-lane branch).
__device__ __forceinline__ void warp_umma(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void warp_umma_ts(uint32_t d, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void warp_commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(smem_u32(bar)) : "memory");
}

// 32 lanes x 64 columns of 32-bit TMEM -> 64 registers a thread, both loads in flight before the wait (which sits in
// the same statement, like the library's other TMEM loads).
__device__ __forceinline__ void tmem_ld_x64(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31"
      "}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr), "r"(taddr + 32));
}

// Four lanes exchange their four uint4: lane i of them has the i-th of each lane's afterwards, v[k] from lane k.
__device__ __forceinline__ void transpose4(uint4 (&v)[4], int lane) {
#pragma unroll
  for (int b = 1; b <= 2; b <<= 1) {
    const bool up = lane & b;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k & b) continue;
      uint32_t* lo = &v[k].x;
      uint32_t* hi = &v[k | b].x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t get = __shfl_xor_sync(0xffffffffu, up ? lo[i] : hi[i], b);
        if (up) lo[i] = get;
        else hi[i] = get;
      }
    }
  }
}
// the k-th of the four lanes' rows (null: not to be stored)
__device__ __forceinline__ uint8_t* shared_row(void* row, bool valid, int k, int lane) {
  return reinterpret_cast<uint8_t*>(
      __shfl_sync(0xffffffffu, valid ? reinterpret_cast<unsigned long long>(row) : 0ull, (lane & ~3) | k));
}

template <int D>
__global__ void __launch_bounds__(WIDE_THREADS, 1)
paged_wide_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const AttnArgs a) {
  using C = WCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;                       // [2 pieces][2 row tiles][TQ]
  uint8_t* ring = sQ + 4 * C::TQ;           // [ST][TT]
  WidePiece* pieces = reinterpret_cast<WidePiece*>(ring + C::ST * C::TT);
  uint64_t* full = reinterpret_cast<uint64_t*>(pieces + 2);
  uint64_t* empty = full + C::ST;
  uint64_t* q_full = empty + C::ST;         // [2]
  uint64_t* q_empty = q_full + 2;           // [2]
  uint64_t* s_full = q_empty + 2;           // [2 row tiles][2 buffers]
  uint64_t* p_full = s_full + 4;            // [2][2]
  // [2][2] a P V has completed: one barrier a buffer, as a warp may see two complete between two looks (the scores
  // of tile j say that P V of j - 2 has)
  uint64_t* o_full = p_full + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (misaligned(smem)) {  // uniform across the CTA; nothing allocated yet
    if (threadIdx.x == 0) dt_set_error(DT_ERR_BAD_ARG, 740);
    return;
  }
  Header& head = *reinterpret_cast<Header*>(const_cast<int*>(abort_flag) + 1);
  if (a.wide_first) pdl_wait();
  pdl_next();
  if (!head.load(a, D)) {
    if (threadIdx.x == 0 && blockIdx.x == 0) dt_report(DT_ERR_BAD_ARG, 741);
    pdl_wait();
    return;
  }
  const int W = head[H_W + WIDE], per = head[H_PER + WIDE], E = head[H_E + WIDE];
  const Entry* ent = plan_entries(const_cast<int*>(a.plan), a.G + a.B, a.B, WIDE, a.max_stream);
  const long long x0l = (long long)blockIdx.x * per;
  if (x0l >= W) {
    pdl_wait();
    return;
  }
  const int x0 = (int)x0l, x1 = min(W, x0 + per);
  const int gsz = a.nh / a.nkv, tpt = 128 / gsz;  // tokens of a 128-row tile

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 2);  // both MMA warps
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 2 + 8);  // both MMA warps have issued its scores, the softmax warps have read the record
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (warp == 0) {
    // ───── producer ─────
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    const int P = 1 << a.shift;
    const int box_rows = min(P, BKV), boxes = BKV / box_rows, bsh = __ffs(boxes) - 1;
    const int copies = boxes == 1 ? 1 : boxes * (D / 64);
    const int none = a.pages * a.nkv * P;  // a row past the cache: the box is filled with zeros
    int e = find_entry(ent, E, x0, lane);
    int n = 0, pc = 0;  // ring loads, pieces
    bool ok = true;
    for (int x = x0; x < x1 && ok;) {
      const Entry en = load_entry(ent + e);
      const Piece pi = piece_at(en, x, x1, a.start[WIDE]);
      const int h = pi.h, t0 = pi.t0, t1 = pi.t1, first = x;
      x = pi.next;
      if (x < x1 && x >= en.cum + (en.tiles + a.start[WIDE]) * a.nkv) {  // on to the next entry with tiles
        ++e;
        while (e + 1 < E && __ldcg(&ent[e].tiles) == 0) ++e;
      }
      if (t1 <= t0) continue;
      const int two = en.ntok > tpt ? 2 : 1, b = pc & 1;
      if (pc >= 2) ok = warp_wait(&q_empty[b], ((pc >> 1) & 1) ^ 1, DT_ERR_TIMEOUT_EMPTY, 742, abort_flag, lane);
      if (!ok) break;
      if (lane == 0) {
        WidePiece d;
        d.tiles = t1 - t0;
        d.key0 = t0 * BKV;
        d.keys = en.keys;
        d.vis = en.vis;
        d.causal = en.seg >= a.G;
        d.tok0 = en.tok0;
        d.ntok = en.ntok;
        d.head0 = h * gsz;
        d.direct = a.G == 0 && t0 == 0 && t1 == en.tiles;
        d.pad = 0;
        d.part = piece_row(a, head, WIDE, en, h, blockIdx.x, first, per);
        pieces[b] = d;
        mbar_arrive_expect_tx(&q_full[b], two * tpt * gsz * 128 * (D / 64));
        for (int u = 0; u < two; ++u)
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_load_3d(sQ + (b * 2 + u) * C::TQ + c * (128 * 128), &tmQ, &q_full[b], c * 64, h * gsz, en.tok0 + u * tpt);
      }
      ++pc;
      const int* table = en.seg < a.G ? a.prefix_tables + en.seg * a.ld_prefix
                                      : a.tables + (en.seg - a.G) * a.ld_tables;
      int win0 = -1, win = 0;  // 32 page ids of the table, one a lane
      // the order of use: K0 K1 V0 K2 V1 ... V(nt - 1), from t0; step i loads K(i) and V(i - 1). Lane c * boxes + b fetches
      // 64-column chunk c of box b; a page that holds the whole tile is one copy with both chunks in it.
      auto load = [&](const CUtensorMap* map, int row, int site) {
        const int st = n % C::ST;
        if (n >= C::ST) ok = warp_wait(&empty[st], ((n / C::ST) & 1) ^ 1, DT_ERR_TIMEOUT_EMPTY, site, abort_flag, lane);
        if (!ok) return;
        if (lane == 0) mbar_arrive_expect_tx(&full[st], C::TT);
        __syncwarp();
        if (lane < copies)
          tma_load_3d(ring + st * C::TT + (lane >> bsh) * (BKV * 128) + (lane & (boxes - 1)) * box_rows * 128, map,
                      &full[st], 0, row, lane >> bsh);
        __syncwarp();
        ++n;
      };
      int row = none, row_v = none;
      for (int t = t0; t <= t1 && ok; ++t) {
        if (t < t1) {
          const int k0 = t * BKV, p0 = k0 >> a.shift, p1 = (min(k0 + BKV, en.keys) - 1) >> a.shift;
          if (win0 < 0 || p1 >= win0 + 32) {
            win0 = p0;
            const int p = win0 + lane;
            win = p * P < en.keys ? __ldcg(table + p) : 0;
            if (p * P < en.keys && (unsigned)win >= (unsigned)a.pages) {
              dt_report(DT_ERR_BOUNDS, 743);
              win = -1;
            }
          }
          const int key = k0 + (lane & (boxes - 1)) * box_rows;
          const int page = __shfl_sync(0xffffffffu, win, ((key >> a.shift) - win0) & 31);
          row_v = row;
          row = key < en.keys && page >= 0 ? (page * a.nkv + h) * P + (key & (P - 1)) : none;
          load(&tmK, row, 744);
        } else {
          row_v = row;
        }
        if (ok && t > t0) load(&tmV, row_v, 749);
      }
    }
    if (ok && pc >= 2)
      ok = warp_wait(&q_empty[pc & 1], ((pc >> 1) & 1) ^ 1, DT_ERR_TIMEOUT_EMPTY, 757, abort_flag, lane);
    if (ok && lane == 0) {
      pieces[pc & 1].tiles = 0;
      mbar_arrive(&q_full[pc & 1]);
    }
    // no load may be in flight into shared memory when the CTA ends, not after an aborted run either (bounded)
    if (lane == 0) {
      const uint64_t w0 = dt_globaltimer();
      for (int k = max(0, n - C::ST); k < n; ++k)
        while (!mbar_try_wait(&full[k % C::ST], (k / C::ST) & 1) && dt_globaltimer() - w0 < 20000000ull) {}
      // (behind the end mark the slot before the last has been released; without it neither has moved on)
      for (int k = max(0, pc - (ok ? 1 : 2)); k < pc; ++k)
        while (!mbar_try_wait(&q_full[k & 1], (k >> 1) & 1) && dt_globaltimer() - w0 < 20000000ull) {}
    }
  } else if (warp <= 2) {
    // ───── MMA of row tile u: the whole warp runs the loop, one elected lane issues ─────
    constexpr uint32_t idS = umma_idesc_bf16(128, BKV, 0, 0), idO = umma_idesc_bf16(128, D, 0, 1);
    const int u = warp - 1;
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t tS = tm + C::C_S + u * 128, tO = tm + C::C_O + u * D;
    const uint64_t dQ0 = umma_smem_desc_sw128(smem_u32(sQ + u * C::TQ), 16, 1024);
    uint64_t dQ = dQ0;
    const uint64_t dK = umma_smem_desc_sw128(smem_u32(ring), 16, 1024);
    const uint64_t dV = umma_smem_desc_sw128(smem_u32(ring), BKV * 128, 1024);
    constexpr uint64_t STG = (uint64_t)(C::TT >> 4);
    int st = 0, par = 0;          // stage and parity of the next ring tile
    int sn = 0, vn = 0;           // S and P V issued: their parity is the buffer
    bool ok = true, issued = false;
    // the next ring tile: waits for it and returns its stage
    auto next = [&](int site) -> int {
      ok = warp_wait(&full[st], par, DT_ERR_TIMEOUT_FULL, site, abort_flag, lane);
      const int at = st;
      if (++st == C::ST) {
        st = 0;
        par ^= 1;
      }
      return at;
    };
    auto score = [&](int at) {  // S = Q K^T of the K tile in stage `at`
      tc_fence_after();
      const uint64_t k = dK + (uint64_t)at * STG;
      const uint32_t d = tS + (sn & 1) * 64;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) warp_umma(d, dQ + qoff(c), k + koff(c), idS, c > 0 ? 1u : 0u);
      warp_commit(&s_full[u * 2 + (sn & 1)]);
      warp_commit(&empty[at]);
      ++sn;
      issued = true;
    };
    for (int pc = 0; ok; ++pc) {
      const int b = pc & 1;
      ok = warp_wait(&q_full[b], (pc >> 1) & 1, DT_ERR_TIMEOUT_FULL, 745, abort_flag, lane);
      if (!ok) break;
      const int nt = __shfl_sync(0xffffffffu, pieces[b].tiles, 0);
      if (nt == 0) break;
      const bool mine = u == 0 || __shfl_sync(0xffffffffu, (int)(pieces[b].ntok > tpt), 0) != 0;
      dQ = dQ0 + (uint64_t)(b * (2 * C::TQ >> 4));
      if (!mine) {  // a piece of one row tile: the other MMA warp releases the ring's tiles as they come
        warp_commit(&q_empty[b]);
        for (int j = 0; j < 2 * nt && ok; ++j) {
          const int at = next(746);
          if (ok) warp_commit(&empty[at]);
        }
        continue;
      }
      for (int j = 0; j < nt && j < 2; ++j) {
        const int ak = next(747);
        if (!ok) break;
        score(ak);
      }
      if (!ok) break;
      if (nt <= 2) warp_commit(&q_empty[b]);
      for (int j = 0; j < nt; ++j) {
        const int av = next(748);
        if (!ok) break;
        ok = warp_wait(&p_full[u * 2 + (vn & 1)], (vn >> 1) & 1, DT_ERR_TIMEOUT_TMEM, 756, abort_flag, lane);
        if (!ok) break;
        tc_fence_after();
        const uint64_t v = dV + (uint64_t)av * STG;
        const uint32_t p = tS + (vn & 1) * 64;
#pragma unroll
        for (int c = 0; c < BKV / 16; ++c) warp_umma_ts(tO, p + c * 8, v + voff(c), idO, (j > 0 || c > 0) ? 1u : 0u);
        warp_commit(&o_full[u * 2 + (vn & 1)]);
        warp_commit(&empty[av]);
        ++vn;
        if (j + 2 < nt) {
          const int ak = next(755);
          if (!ok) break;
          score(ak);
          if (j + 3 == nt) warp_commit(&q_empty[b]);
        }
      }
    }
    if (!ok && issued) {  // let the products already issued finish before TMEM is freed (bounded)
      const uint64_t w0 = dt_globaltimer();
      while (dt_globaltimer() - w0 < 2000000ull) {}
    }
  } else if (warp >= 4) {
    // ───── softmax: row r of tile u = TMEM lane r ─────
    const int u = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t tS = tmem + C::C_S + u * 128 + lane_off, tO = tmem + C::C_O + u * D + lane_off;
    const float sl2 = a.scale * LOG2E_F;
    const uint64_t sl2v = f2_pack(sl2, sl2);
    int sn = 0, n = 0;  // key tiles of this row tile, ring position
    bool ok = true;
    for (int pc = 0; ok; ++pc) {
      ok = warp_wait(&q_full[pc & 1], (pc >> 1) & 1, DT_ERR_TIMEOUT_FULL, 759, abort_flag, lane);
      if (!ok) break;
      const WidePiece en = pieces[pc & 1];
      __syncwarp();
      if (en.tiles == 0) break;
      if (lane == 0) mbar_arrive(&q_empty[pc & 1]);
      if (u == 0 || en.ntok > tpt) {
        const int tok = u * tpt + r / gsz, hh = r % gsz;
        const bool valid = r < tpt * gsz && tok < en.ntok;
        // (rows of no token are computed like the others and left out at the end)
        const int vis = valid ? min(en.vis + (en.causal ? tok : 0), en.keys) : en.keys;
        float m = -INFINITY, l = 0.f;
        for (int j = 0; j < en.tiles; ++j, ++sn) {
          const int buf = sn & 1;
          ok = warp_wait(&s_full[u * 2 + buf], (sn >> 1) & 1, DT_ERR_TIMEOUT_TMEM, 750, abort_flag, lane);
          if (!ok) break;
          tc_fence_after();
          uint32_t sv[64];
          tmem_ld_x64(tS + buf * 64, sv);
          const int k0 = en.key0 + j * BKV, hi = vis - k0;  // columns e < hi are seen
          if (en.keys - k0 < BKV) {  // the segment's last tile: zero the V rows behind its last key (each row tile for itself)
            const int nt = en.tiles, vs = n + min(nt, 2) + j + min(j, max(nt - 2, 0)), gone = en.keys - k0;
            ok = warp_wait(&full[vs % C::ST], (vs / C::ST) & 1, DT_ERR_TIMEOUT_FULL, 751, abort_flag, lane);
            if (!ok) break;
            uint4* v = reinterpret_cast<uint4*>(ring + (vs % C::ST) * C::TT);
            for (int c = 0; c < D / 64; ++c)
              for (int i = gone * 8 + quad * 32 + lane; i < BKV * 8; i += 128) v[c * (BKV * 8) + i] = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
          }
          if (__any_sync(0xffffffffu, hi < BKV)) {
#pragma unroll
            for (int i = 0; i < 64; ++i) sv[i] = i < hi ? sv[i] : 0xff800000u;
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(sv[i]));
          const float mn = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;  // -inf: nothing seen yet
          bool resc = false;
          float mo = m;
          if (mn > m + RESCALE_THRESHOLD || m == -INFINITY) {
            resc = m != -INFINITY;
            m = mn;
          }
          if (__any_sync(0xffffffffu, resc)) {
            ok = warp_wait(&o_full[u * 2 + ((sn - 1) & 1)], ((sn - 1) >> 1) & 1, DT_ERR_TIMEOUT_TMEM, 754, abort_flag, lane);
            if (!ok) break;
            tc_fence_after();
            const float al = resc ? ex2_approx(mo - m) : 1.f;
            l *= al;
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(tO + c, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * al);
              tmem_st_32x32b_x16(tO + c, o);
            }
          }
          // P goes to the tensor cores in bf16, half a step 2^-8 each. The sum takes the values before that: their roundings
          // cancel over the keys as they do in the products (random scores: 2.29e-3 of the output's norm off either way at
          // 4000 keys; weights that are all alike share one rounding, so then up to 2^-8 of the output), and the rounded
          // ones would have to be unpacked again for every pair.
          const float ms = m == -INFINITY ? 0.f : m;
          const uint64_t nm = f2_pack(-ms, -ms);
          uint64_t sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            const float2 y = f2_unpack(f2_fma(f2_pack(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1])), sl2v, nm));
            const float p0 = ex2_approx(y.x), p1 = ex2_approx(y.y);
            sum[(i >> 1) & 1] = f2_add(sum[(i >> 1) & 1], f2_pack(p0, p1));
            pk[i / 2] = pack_bf16(p0, p1);
          }
          tmem_st_32x32b_x32(tS + buf * 64, pk);
          const float2 s2 = f2_unpack(f2_add(sum[0], sum[1]));
          l += s2.x + s2.y;
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[u * 2 + buf]);
        }
        if (ok) ok = warp_wait(&o_full[u * 2 + ((sn - 1) & 1)], ((sn - 1) >> 1) & 1, DT_ERR_TIMEOUT_TMEM, 752, abort_flag, lane);
        if (!ok) break;
        tc_fence_after();
        const float inv = l != 0.f ? 1.f / l : 0.f;  // (nothing seen: zeros; a NaN goes on)
        const float ls = l != 0.f ? m + log2f(l) : -INFINITY;
        const bool direct = en.direct;
        const long long row = (long long)(en.tok0 + tok) * a.nh + en.head0 + hh;
        const long long part = en.part + tok * gsz + hh;
        // 64 bytes of a row a lane, exchanged between four lanes: a store then covers eight rows' 64 bytes instead of
        // 16 bytes of 32 rows, which the load-store unit takes one row a clock
        if (direct) {
          uint8_t* rows[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) rows[k] = shared_row(a.out + row * D, valid, k, lane);
#pragma unroll 1  // (straight code of this length waits for its instructions)
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(tO + c, o);
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t* w = &v[i].x;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                w[k] = l != 0.f ? pack_bf16(__uint_as_float(o[8 * i + 2 * k]) * inv, __uint_as_float(o[8 * i + 2 * k + 1]) * inv) : 0u;
            }
            transpose4(v, lane);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (rows[k]) *reinterpret_cast<uint4*>(rows[k] + c * 2 + (lane & 3) * 16) = v[k];
          }
        } else {
          uint8_t* rows[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) rows[k] = shared_row(a.part_o + part * D, valid, k, lane);
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(tO + c, o);
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 16; ++i) (&v[i / 4].x)[i % 4] = l != 0.f ? __float_as_uint(__uint_as_float(o[i]) * inv) : 0u;
            transpose4(v, lane);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (rows[k]) *reinterpret_cast<uint4*>(rows[k] + c * 4 + (lane & 3) * 16) = v[k];
          }
        }
        if (valid) {
          if (!direct) a.part_lse[part] = ls;
          else if (a.lse) a.lse[row] = ls * LN2_F;
        }
        tc_fence_before();
      }
      n += 2 * en.tiles;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, C::TMEM_COLS);
  pdl_wait();
}

// ───────────────────────── join of the pieces ─────────────────────────
// One warp a (token, head): its prefix pieces and its own pieces, weighted by 2^(lse - max). With groups a block
// takes eight heads of one token, or all heads of two tokens where there are many; a warp a token looks up where its
// pieces lie, for all heads at once, before the kernels in front of this one have finished. Without, only items cut by
// a CTA boundary have pieces to join (all others went straight to `out`): a block takes one boundary and 16 or
// JOIN_ROWS rows, if the boundary is the item's first. Rows that see nothing are zeroed. Bound: the latency of a row's
// loads, which do not wait for each other, and with many rows the instructions of each. It adds 4.5 us to one token's
// call, 4 us to a decode step of 64 requests, 7 us to 128 answers, 13 us to 1214 scored tokens. (Left to the CTA that finishes an
// item's last piece, the same join cost one token 4 us more: its code comes in cold, behind an atomic.)
constexpr int JOIN_THREADS = 256, JOIN_HEADS = 32;  // threads, kv heads of a block at most
constexpr int JOIN_ROWS = 64;  // rows of a WIDE boundary a block (a prompt part: 16 338 us, 32 335, 64 328, 128 348)

// The pieces of an item: CTAs c0 .. c0 + count - 1 of its line, from the first that has a key tile of it. `lane`
// + k0 picks one; its partial result's row for row r of the item.
struct Pieces {
  int which, h, c0, count, x0, per;
  Entry en;
  __device__ long long row(const AttnArgs& a, const Header& head, int i, int r) const {
    const int c = c0 + i;
    return piece_row(a, head, which, en, h, c, max(x0, c * per), per) + r;
  }
};
__device__ __forceinline__ Pieces pieces_of(const AttnArgs& a, const Header& head, int which, const Entry& en, int h) {
  const int start = a.start[which];
  Pieces p;
  p.which = which;
  p.h = h;
  p.per = head[H_PER + which];
  p.x0 = en.cum + h * (en.tiles + start);
  p.c0 = (p.x0 + start) / p.per;
  p.count = en.tiles > 0 ? (p.x0 + start + en.tiles - 1) / p.per - p.c0 + 1 : 0;
  p.en = en;
  return p;
}

// Joins `total` pieces of a row, the i-th at row_of(i), and writes the row of `out`: up to 32 pieces a turn, one a lane
// for their log-sum-exp, then their rows, whose loads do not wait for each other.
template <int D, typename F>
__device__ __forceinline__ void join_row(const AttnArgs& a, int total, F&& row_of, long long out_row, int lane) {
  constexpr int K = (D + 31) / 32;  // columns of a lane, side by side
  using V = std::conditional_t<K == 4, float4, std::conditional_t<K == 2, float2, float>>;
  const bool on = D >= 32 || lane < D;
  float m = -INFINITY, l = 0.f, acc[K] = {};
  for (int k0 = 0; k0 < total; k0 += 32) {
    const int n = min(32, total - k0);
    long long row = 0;
    float ls = -INFINITY;
    if (lane < n) {
      row = row_of(k0 + lane);
      ls = __ldcg(a.part_lse + row);
    }
    if (__all_sync(0xffffffffu, ls == -INFINITY)) continue;  // (a NaN is no such piece)
    const float mn = fmaxf(m, warp_max(ls)), ms = mn == -INFINITY ? 0.f : mn;
    const float f = ex2_approx(m - ms), w = ex2_approx(ls - ms);
    m = mn;
    l = l * f + warp_sum(w);
#pragma unroll
    for (int k = 0; k < K; ++k) acc[k] *= f;
    for (int j0 = 0; j0 < n; j0 += 4) {
      V v[4];
      float wj[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        wj[j] = __shfl_sync(0xffffffffu, w, j0 + j);  // (lanes of no piece weigh nothing)
        const float* o = a.part_o + __shfl_sync(0xffffffffu, row, j0 + j) * D + lane * K;
        v[j] = V{};
        if (on && wj[j] != 0.f) v[j] = __ldcg(reinterpret_cast<const V*>(o));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int k = 0; k < K; ++k) acc[k] += wj[j] * reinterpret_cast<const float*>(&v[j])[k];
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  __nv_bfloat16* o = a.out + out_row * D + lane * K;
  if constexpr (K == 4)
    *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv));
  else if constexpr (K == 2)
    *reinterpret_cast<uint32_t*>(o) = pack_bf16(acc[0] * inv, acc[1] * inv);
  else if (on)
    *o = __float2bfloat16(acc[0] * inv);
  if (a.lse && lane == 0) a.lse[out_row] = l != 0.f ? (m + log2f(l)) * LN2_F : -INFINITY;
}

// last i in [0, n) with v[i] <= x; a decode step's token t is request t's, which is tried first, then 32 probes a round
__device__ __forceinline__ int find_last(const int* v, int n, int x, int lane) {
  if (x < n && __ldcg(v + x) == x && __ldcg(v + x + 1) == x + 1) return x;
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const unsigned m = __ballot_sync(0xffffffffu, at < hi && __ldcg(v + at) <= x);
    const int nlo = lo + (31 - __clz(m | 1u)) * step;
    hi = min(hi, nlo + step);
    lo = nlo;
  }
  return lo;
}

template <int D>
__global__ void __launch_bounds__(JOIN_THREADS, 4)
paged_join_kernel(const AttnArgs a, int tpt0, int tpt1, int tokens, int heads) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = JOIN_THREADS / 32;
  __shared__ Header head;
  __shared__ Entry s_entry;
  __shared__ int s_go;
  __shared__ long long s_row[2][2][JOIN_HEADS];  // a token's pieces in its prefix and its own segment: the first's row
  __shared__ int s_count[2][2][JOIN_HEADS], s_tile[2][2];  // for the kv head's first query head, how many, rows apart
  const bool fits = head.load(a, D) && head[H_STATUS] == 0;
  const int N = head[H_N], gsz = a.nh / a.nkv;
  const int* seg_first = a.plan + H_INTS;
  const int* group_of = plan_requests(const_cast<int*>(a.plan), a.G + a.B);
  auto entries = [&](int which) {
    return plan_entries(const_cast<int*>(a.plan), a.G + a.B, a.B, which, a.max_stream);
  };
  bool waited = false;  // everything up to the first partial result comes from the plan, before this kernel's turn
  auto wait = [&] {
    if (!waited) pdl_wait();
    waited = true;
  };
  // the entry of token t in segment s (one without tiles if there is none), by one warp
  auto look_up = [&](int s, int t, int tok0, int& which) {
    const int f = __ldcg(seg_first + s);
    which = f >= 0 && (f & WIDE_BIT) ? WIDE : STREAM;
    Entry e{};
    if (f >= 0) e = load_entry(entries(which) + (f & ~WIDE_BIT) + (t - tok0) / (which ? tpt1 : tpt0));
    return e;
  };
  if (fits && a.G == 0) {
    // 16 rows of a STREAM boundary, JOIN_ROWS of a WIDE one
    const int W0 = head[H_W], W1 = head[H_W + 1], per0 = head[H_PER], per1 = head[H_PER + 1];
    const int cuts0 = W0 ? (W0 - 1) / per0 : 0, cuts1 = W1 ? (W1 - 1) / per1 : 0;
    constexpr int PARTS = WIDE_ROWS / JOIN_ROWS;
    for (int k = blockIdx.x; k < cuts0 + PARTS * cuts1; k += gridDim.x) {
      const int which = k < cuts0 ? STREAM : WIDE, per = which ? per1 : per0;
      const int c = (which ? (k - cuts0) / PARTS : k) + 1, r0 = which ? (k - cuts0) % PARTS * JOIN_ROWS : 0;
      const int x = c * per;
      if (warp == 0) {
        const Entry* ent = entries(which);
        const Entry e = load_entry(ent + find_entry(ent, head[H_E + which], x, lane));
        if (lane == 0) s_entry = e;
      }
      __syncthreads();
      const Entry en = s_entry;
      const int start = a.start[which], units = en.tiles + start, h = (x - en.cum) / units, x0 = en.cum + h * units;
      if (x > x0 + start && (x0 + start) / per + 1 == c) {
        wait();
        const Pieces p = pieces_of(a, head, which, en, h);
        for (int r = r0 + warp; r < min(r0 + (which ? JOIN_ROWS : STREAM_ROWS), en.ntok * gsz); r += nw) {
          const int tok = r / gsz;
          join_row<D>(a, p.count, [&](int i) { return p.row(a, head, i, r); },
                      (long long)(en.tok0 + tok) * a.nh + h * gsz + (r - tok * gsz), lane);
        }
      }
      __syncthreads();  // the entry is read before the next one is put there
    }
    if (head[H_EMPTY] != 0) {
      wait();
      for (int t = blockIdx.x; t < N; t += gridDim.x) {
        if (warp == 0) {
          const int i = find_last(a.cu_q, a.B, t, lane);
          int which;
          const Entry en = look_up(i, t, __ldcg(a.cu_q + i), which);
          if (lane == 0) s_go = en.ntok == 0 || en.vis + (t - en.tok0) <= 0;
        }
        __syncthreads();
        if (s_go)
          for (int h = warp; h < a.nh; h += nw)
            join_row<D>(a, 0, [](int) { return 0ll; }, (long long)t * a.nh + h, lane);
        __syncthreads();
      }
    }
  } else if (fits) {
    const int chunks = (a.nh + heads - 1) / heads, blocks = (N + tokens - 1) / tokens * chunks;
    for (int k = blockIdx.x; k < blocks; k += gridDim.x) {
      const int t0 = k / chunks * tokens, hd0 = (k - k / chunks * chunks) * heads, t = t0 + warp;
      const int h0 = hd0 / gsz, nt = min(tokens, N - t0), nd = min(heads, a.nh - hd0);
      if (warp < nt) {
        const int i = find_last(a.cu_q, a.B, t, lane), y = __ldcg(group_of + i);
        const int tok0[2] = {__ldcg(a.cu_q + __ldcg(a.cu_group + y)), __ldcg(a.cu_q + i)};
#pragma unroll
        for (int own = 0; own < 2; ++own) {
          int which;
          const Entry en = look_up(own ? a.G + i : y, t, tok0[own], which);
          const int h = h0 + lane;
          if (h < a.nkv && lane < JOIN_HEADS) {
            const Pieces p = pieces_of(a, head, which, en, h);
            s_row[warp][own][lane] = p.row(a, head, 0, (t - en.tok0) * gsz);
            s_count[warp][own][lane] = p.count;
          }
          if (lane == 0) s_tile[warp][own] = which ? WIDE_ROWS : STREAM_ROWS;
        }
      }
      __syncthreads();
      wait();
      for (int r = warp; r < nt * nd; r += nw) {
        const int j = r >= nd, hd = hd0 + r - j * nd, h = hd / gsz, x = hd - h * gsz;
        const int np = s_count[j][0][h - h0], total = np + s_count[j][1][h - h0];
        const long long rp = s_row[j][0][h - h0] + x, rq = s_row[j][1][h - h0] + x;
        const int tp = s_tile[j][0], tq = s_tile[j][1];
        // (the pieces of an item lie a tile of rows apart)
        join_row<D>(a, total, [&](int i) { return i < np ? rp + i * tp : rq + (i - np) * tq; },
                    (long long)(t0 + j) * a.nh + hd, lane);
      }
      __syncthreads();
    }
  }
  wait();  // a kernel after this one may rely on the ones before it
}

// ───────────────────────── host ─────────────────────────
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;

bool have_encode() {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  return g_encode != nullptr;
}

CUtensorMapSwizzle swizzle_of(int columns) {
  return columns == 64 ? CU_TENSOR_MAP_SWIZZLE_128B
         : columns == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
}

// [pages * nkv * page_size rows][D] bf16, boxes of `rows` rows of up to 64 columns
int cache_map(CUtensorMap* m, const void* base, long long total_rows, int D, int rows) {
  if (!have_encode()) return -2;
  const int cw = D < 64 ? D : 64;
  cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)total_rows};
  cuuint64_t strides[1] = {(cuuint64_t)D * 2};
  cuuint32_t box[2] = {(cuuint32_t)cw, (cuuint32_t)rows};
  cuuint32_t estr[2] = {1, 1};
  return g_encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle_of(cw), CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -3;
}

// the cache for the WIDE kernel: [d / 64][row][64 columns], boxes of `rows` rows; a box of a whole tile has all its
// column chunks
int chunked_map(CUtensorMap* m, const void* base, long long total_rows, int D, int rows) {
  if (!have_encode()) return -2;
  const cuuint64_t dims[3] = {64, (cuuint64_t)total_rows, (cuuint64_t)(D / 64)};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, 128};
  const cuuint32_t box[3] = {64, (cuuint32_t)rows, (cuuint32_t)(rows == BKV ? D / 64 : 1)};
  const cuuint32_t estr[3] = {1, 1, 1};
  return g_encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -3;
}

// q [T][nh][D]: boxes of `tpt` tokens x one kv group's heads x up to 64 columns
int query_map(CUtensorMap* m, const void* base, int T, int nh, int D, int gsz, int tpt) {
  if (!have_encode()) return -2;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)nh, (cuuint64_t)T};
  cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)nh * D * 2};
  const int cw = D < 64 ? D : 64;
  cuuint32_t box[3] = {(cuuint32_t)cw, (cuuint32_t)gsz, (cuuint32_t)tpt};
  cuuint32_t estr[3] = {1, 1, 1};
  return g_encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle_of(cw), CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -3;
}

// What is asked of a device once: its SM count, and the kernels' shared memory limits (see prepared()).
constexpr int MAX_DEVICES = 64;
std::atomic<int> g_sms[MAX_DEVICES];
int sm_count(int* sms, int* device = nullptr) {
  int dev = 0;
  DT_CUDA_RET(cudaGetDevice(&dev));
  if (dev >= MAX_DEVICES) return -12;
  if (device) *device = dev;
  *sms = g_sms[dev].load(std::memory_order_relaxed);
  if (*sms == 0) {
    DT_CUDA_RET(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
    g_sms[dev].store(*sms, std::memory_order_relaxed);
  }
  return 0;
}
template <typename K>
int prepared(K* kernel, int smem, std::atomic<bool> (&done)[MAX_DEVICES], int device) {
  if (done[device].load(std::memory_order_acquire)) return 0;
  DT_CUDA_RET(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  done[device].store(true, std::memory_order_release);
  return 0;
}

// An item's start and end in key tiles (of 32 or 64 and of 64 keys). STREAM: 64 requests of up to 4096 keys take
// 67.4 / 66.5 / 65.9 / 65.9 / 66.0 / 66.5 us with 0 / 1 / 2 / 3 / 4 / 6, 200 requests of up to 300 keys 23.8 / 22.7 / 22.6 /
// 22.7 / 22.6 / 23.6. WIDE: 60 questions' answers over shared pages take
// 40.5 / 41.7 / 42.6 / 44.4 us and a prompt's second part 340 / 338 / 341 / 343 us with 2 / 3 / 4 / 6.
constexpr int START_STREAM = 3, START_WIDE = 2;

// What a batch shape implies for both kernels.
struct Shape {
  int T, B, G, nh, nkv, d, gsz, sms, device;
  bool wide, wide_first;          // whether WIDE segments can occur, which kernel goes first
  int tpt[2], kt[2], ctas[2], max_entries[2], start[2];
  long long part_rows;
};
int shape_of(Shape* s, int T, int B, int G, int nh, int nkv, int d) {
  if (T < 0 || T > (1 << 24) || B < 1 || B > 8192 || G < 0 || G > B || nkv < 1 || nh < nkv || nh % nkv ||
      nh / nkv > STREAM_ROWS || (long long)T * nh >= (1 << 29) || (d != 16 && d != 32 && d != 64 && d != 128))
    return -10;
  const int rc = sm_count(&s->sms, &s->device);
  if (rc) return rc;
  s->T = T; s->B = B; s->G = G; s->nh = nh; s->nkv = nkv; s->d = d; s->gsz = nh / nkv;
  s->wide = d >= 64 && (long long)T * s->gsz > STREAM_ROWS;
  // A step of about one token a request has nothing for WIDE: in front, its blocks are gone before STREAM's need the
  // shared memory, and the join starts right behind STREAM (64 requests: 67.2 -> 63.7 us). Where WIDE has work it goes
  // second, and starts on the SMs that STREAM leaves (in front: answers 36.0 -> 38.2 us, a prompt part 333 -> 339).
  s->wide_first = s->wide && G == 0 && T <= 2 * B;
  s->tpt[STREAM] = STREAM_ROWS / s->gsz;
  s->tpt[WIDE] = 2 * (128 / s->gsz);
  s->kt[STREAM] = d == 128 ? DCfg<128>::KT : DCfg<64>::KT;
  s->kt[WIDE] = BKV;
  s->ctas[STREAM] = DEC_CTAS * s->sms;
  s->ctas[WIDE] = s->sms;
  s->start[STREAM] = START_STREAM;
  s->start[WIDE] = START_WIDE;
  const int times = G ? 2 : 1;  // a token is in its request's segment and its group's
  s->max_entries[STREAM] = G + B + (d < 64 ? times * (T / s->tpt[STREAM]) : 0);
  s->max_entries[WIDE] = s->wide ? G + B + times * (T / s->tpt[WIDE]) : 0;
  const long long stream = (long long)s->ctas[STREAM] * STREAM_ROWS, wide = s->wide ? (long long)s->ctas[WIDE] * WIDE_ROWS : 0;
  s->part_rows = G ? 2LL * T * nh + stream + wide : 2 * (stream + wide);
  return 0;
}

long long plan_bytes(const Shape& s) {
  return (long long)(H_INTS + (s.G + s.B + 7) / 8 * 8 + (s.B + 7) / 8 * 8) * 4 +
         ((long long)s.max_entries[STREAM] + s.max_entries[WIDE]) * (long long)sizeof(Entry);
}
long long work_bytes(const Shape& s) { return s.part_rows * (s.d + 1) * 4; }

// launch that may begin while the kernel before it in the stream still runs (see pdl_wait)
template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), int grid, int threads, int smem, cudaStream_t st, const A&... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = st;
  c.attrs = &attr;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args...);
}

template <int D>
int attn_launch(const AttnArgs& a, const Shape& s, const void* kc, const void* vc, cudaStream_t st) {
  using C = DCfg<D>;
  const int P = 1 << a.shift;
  const long long rows = (long long)a.pages * a.nkv * P;
  CUtensorMap mq, mk, mv;
  auto wide = [&]() -> int {
    if constexpr (D >= 64) {
      int rc = query_map(&mq, a.q, a.T, a.nh, D, s.gsz, 128 / s.gsz);
      if (!rc) rc = chunked_map(&mk, kc, rows, D, P < BKV ? P : BKV);
      if (!rc) rc = chunked_map(&mv, vc, rows, D, P < BKV ? P : BKV);
      static std::atomic<bool> done[MAX_DEVICES];
      if (!rc) rc = prepared(paged_wide_kernel<D>, WCfg<D>::SMEM, done, s.device);
      if (rc) return rc;
      DT_CUDA_RET(launch_early(paged_wide_kernel<D>, s.ctas[WIDE], WIDE_THREADS, WCfg<D>::SMEM, st, mq, mk, mv, a));
    }
    return 0;
  };
  auto stream = [&]() -> int {
    int rc = query_map(&mq, a.q, a.T, a.nh, D, s.gsz, s.tpt[STREAM]);
    if (!rc) rc = cache_map(&mk, kc, rows, D, P < C::KT ? P : C::KT);
    if (!rc) rc = cache_map(&mv, vc, rows, D, P < C::KT ? P : C::KT);
    static std::atomic<bool> done[MAX_DEVICES];
    if (!rc) rc = prepared(paged_stream_kernel<D>, C::SMEM, done, s.device);
    if (rc) return rc;
    DT_CUDA_RET(launch_early(paged_stream_kernel<D>, s.ctas[STREAM], DEC_THREADS, C::SMEM, st, mq, mk, mv, a));
    return 0;
  };
  int rc = s.wide_first ? wide() : stream();
  if (!rc && s.wide) rc = s.wide_first ? stream() : wide();
  if (rc) return rc;
  // With groups: eight heads of one token a block, or all heads of two tokens where that still fills the GPU (8 or 4
  // tokens a block measured 20 and 3 us more for 1214 scored tokens than two, one 5 us more).
  const int nw = JOIN_THREADS / 32, tokens = a.T >= 4 * s.sms && a.nkv <= JOIN_HEADS ? 2 : 1, heads = tokens == 1 ? nw : a.nh;
  long long blocks = a.G ? (long long)((a.T + tokens - 1) / tokens) * ((a.nh + heads - 1) / heads)
                         : s.ctas[STREAM] + (s.wide ? WIDE_ROWS / JOIN_ROWS * s.ctas[WIDE] : 0);
  if (blocks > 8 * s.sms) blocks = 8 * s.sms;
  return (int)launch_early(paged_join_kernel<D>, (int)blocks, JOIN_THREADS, 0, st, a, s.tpt[STREAM], s.tpt[WIDE], tokens,
                           heads);
}

}  // namespace

// Bytes of the plan and of the scratch buffer for up to T tokens, B requests, G groups (negative: bad shape).
DT_API long long dt_paged_plan_bytes(int T, int B, int G, int nh, int nkv, int d) {
  Shape s;
  const int rc = shape_of(&s, T, B, G, nh, nkv, d);
  if (rc) return rc < 0 ? rc : -1;
  return plan_bytes(s);
}
DT_API long long dt_paged_work_bytes(int T, int B, int G, int nh, int nkv, int d) {
  Shape s;
  const int rc = shape_of(&s, T, B, G, nh, nkv, d);
  if (rc) return rc < 0 ? rc : -1;
  return work_bytes(s);
}
// Kernels that dt_paged_attention launches for a shape.
DT_API int dt_paged_kernels(int T, int B, int G, int nh, int nkv, int d) {
  Shape s;
  return shape_of(&s, T, B, G, nh, nkv, d) ? 0 : s.wide ? 3 : 2;
}

// Arguments of both launchers (pointers and 64-bit values first, then ints, no padding).
struct PagedPlanArgs {
  int* plan;
  const int *cu_q, *lens, *cu_group, *prefix_lens;
  int T, B, G, nh, nkv, d, shift, max_own, max_prefix, reserved;
};
DT_API int dt_paged_plan(const PagedPlanArgs* args, cudaStream_t st) {
  const PagedPlanArgs& g = *args;
  Shape s;
  const int rc = shape_of(&s, g.T, g.B, g.G, g.nh, g.nkv, g.d);
  if (rc) return rc;
  if (g.shift < 4 || g.shift > 7 || !g.plan) return -10;
  PlanArgs a{g.cu_q, g.lens, g.cu_group, g.prefix_lens, g.T, g.B, g.G, g.nh, g.nkv, g.d, g.shift, g.max_own, g.max_prefix,
             s.wide ? STREAM_ROWS : 0x7fffffff, {}, {}, {}, {}, {}};
  for (int w = 0; w < 2; ++w) {
    a.tpt[w] = s.tpt[w];
    a.kt[w] = s.kt[w];
    a.ctas[w] = s.ctas[w];
    a.max_entries[w] = s.max_entries[w];
    a.start[w] = s.start[w];
  }
  // A thread a segment, in as few warps as do it in one turn: the block's barriers and the scan of its warps are the time
  // of a small plan, the turns that of a large one. Plan alone, with 128 / 256 / 1024 threads: 64 requests 3.5 / 3.9 / 7.2
  // us, 200 5.9 / 4.3 / 7.4, 500 10.0 / 7.2 / 8.0, 1000 18.3 / 12.4 / 11.0, 4000 68 / 44 / 33.
  const int threads = g.G + g.B <= 128 ? 128 : g.G + g.B <= 256 ? 256 : PLAN_THREADS;
  paged_plan_kernel<<<1, threads, 0, st>>>(a, g.plan);
  return (int)cudaGetLastError();
}

struct PagedAttentionArgs {
  const void *q, *kc, *vc;
  void* out;
  float* lse;
  const int* plan;
  void* work;
  const int *cu_q, *cu_group, *tables, *prefix_tables;
  long long ld_tables, ld_prefix;
  double scale;
  int T, B, G, nh, nkv, d, shift, pages, width, prefix_width;
};
DT_API int dt_paged_attention(const PagedAttentionArgs* args, cudaStream_t st) {
  const PagedAttentionArgs& g = *args;
  Shape s;
  const int rc = shape_of(&s, g.T, g.B, g.G, g.nh, g.nkv, g.d);
  if (rc) return rc;
  if (g.shift < 4 || g.shift > 7 || g.pages < 1 || !g.plan || !g.work) return -10;
  if ((reinterpret_cast<uintptr_t>(g.q) | reinterpret_cast<uintptr_t>(g.kc) | reinterpret_cast<uintptr_t>(g.vc) |
       reinterpret_cast<uintptr_t>(g.out) | reinterpret_cast<uintptr_t>(g.work) | reinterpret_cast<uintptr_t>(g.plan)) & 15)
    return -11;
  if (g.T == 0) return 0;
  const long long rows = (long long)g.T * g.nh, cache = 2LL * g.pages * g.nkv * g.d << g.shift;
  const Span out[] = {span(g.out, 2 * rows * g.d), span(g.lse, 4 * rows), span(g.work, work_bytes(s))};
  const Span in[] = {span(g.q, 2 * rows * g.d), span(g.kc, cache), span(g.vc, cache), span(g.plan, plan_bytes(s)),
                     span(g.cu_q, 4LL * (g.B + 1)), span(g.cu_group, 4LL * (g.G + 1)),
                     span_rows(g.tables, g.B, 4LL * g.width, 4 * g.ld_tables),
                     span_rows(g.prefix_tables, g.G, 4LL * g.prefix_width, 4 * g.ld_prefix)};
  if (outputs_shared(out, in)) return -13;
  float* po = reinterpret_cast<float*>(g.work);
  const AttnArgs a{reinterpret_cast<const __nv_bfloat16*>(g.q), reinterpret_cast<__nv_bfloat16*>(g.out), g.lse, g.plan,
                   g.tables, g.prefix_tables, g.ld_tables, g.ld_prefix, g.cu_q, g.cu_group, po, po + s.part_rows * g.d,
                   g.T, g.B, g.G, g.nh, g.nkv, g.shift, g.pages, s.max_entries[STREAM], s.ctas[STREAM], s.wide_first,
                   {s.start[STREAM], s.start[WIDE]}, (float)g.scale};
  if (g.d == 16) return attn_launch<16>(a, s, g.kc, g.vc, st);
  if (g.d == 32) return attn_launch<32>(a, s, g.kc, g.vc, st);
  if (g.d == 64) return attn_launch<64>(a, s, g.kc, g.vc, st);
  return attn_launch<128>(a, s, g.kc, g.vc, st);
}
