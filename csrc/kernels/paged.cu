// Paged key/value cache: page tables and slot maps from request lengths, and the append of new K/V rows.
//
// Cache layout: K and V are [pages, nkv, page, d] bf16, so the rows of one kv head in one page are contiguous
// (the unit the attention kernel fetches). A token's slot is page * page_size + offset; slots are 32-bit
// (the host refuses caches of 2^31 tokens or more), every element offset is 64-bit.
#include "common.cuh"
#include "spans.h"
#include <atomic>

namespace {

// ───────────────────────── page tables ─────────────────────────
// Request i holds c tokens in its table row and adds n: have = ceil(c / P) pages are there, need =
// ceil((c + n) / P) - have are taken from the free list in request order (base = running sum of need).
//   table[i][have + k] = free[base + k];  cu[i + 1] = cu[i] + n;  total[i] = c + n
//   token cu[i] + j sits at x = c + j: position start[i] + x, slot page(x) * P + x % P; tokens past the last: -1
// Bound: latency (a few KB to a few hundred KB). One launch: every block repeats the scan over the B lengths
// (they come from L2 after the first block) instead of a scan kernel before the scatter, and the blocks share
// the new table entries and tokens evenly, each finding its request by a search in shared memory.
// All or nothing: with too few free pages, a table too narrow, more tokens than slots or a negative length,
// nothing is taken (table untouched, every slot -1, cu zero, total = cached) and used[1] says why.
// Measured on the GPU: 3.7 us for a decode step of 256 requests, 4.1 us for 64 prompts of up to 2048 tokens.
constexpr int PT_THREADS = 512, PT_MAX_REQUESTS = 8192;
enum : int { PT_POOL = 1, PT_WIDTH = 2, PT_SLOTS = 4, PT_NEGATIVE = 8 };

struct Pair {
  long long a, b;
};
__device__ __forceinline__ Pair warp_scan(Pair v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, v.a, o), b = __shfl_up_sync(0xffffffffu, v.b, o);
    if (lane >= o) {
      v.a += a;
      v.b += b;
    }
  }
  return v;
}

// largest i in [0, n) with v[i] <= x, for v[0] <= x and v not falling
__device__ __forceinline__ int last_le(const int* v, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(PT_THREADS)
page_tables_kernel(const int* __restrict__ cached, const int* __restrict__ fresh, const int* __restrict__ start,
                   const int* __restrict__ free_pages, int n_free, int* __restrict__ tables, long long ld, int width,
                   int* __restrict__ slots, int* __restrict__ positions, int cap, int* __restrict__ cu,
                   int* __restrict__ total, int* __restrict__ used, int B, int shift) {
  extern __shared__ int sh[];
  int* s_cached = sh;          // [B]
  int* s_cu = s_cached + B;    // [B] exclusive sums of the new tokens
  int* s_base = s_cu + B;      // [B] exclusive sums of the new pages
  __shared__ Pair s_warp[PT_THREADS / 32];
  __shared__ int s_err;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int P = 1 << shift;
  if (tid == 0) s_err = 0;
  __syncthreads();
  long long n_sum = 0, p_sum = 0;  // running totals of the chunks before this one
  for (int i0 = 0; i0 < B; i0 += PT_THREADS) {
    const int i = i0 + tid;
    Pair v{0, 0};
    int err = 0;
    if (i < B) {
      const int c = cached[i], n = fresh[i];
      if (c < 0 || n < 0) {
        err = PT_NEGATIVE;
      } else {
        const long long pages = ((long long)c + n + P - 1) >> shift;
        // (lengths near 2^31, which no table row reaches in int32 slots, would wrap in the 32-bit sums below)
        if (pages > width || (long long)c + n > 0x7fffffff - P) err = PT_WIDTH;
        v.a = n;
        v.b = pages - (((long long)c + P - 1) >> shift);
      }
      s_cached[i] = c;
    }
    if (err) atomicOr(&s_err, err);
    const Pair w = warp_scan(v, lane);
    if (lane == 31) s_warp[warp] = w;
    __syncthreads();
    if (warp == 0) {
      Pair t = lane < PT_THREADS / 32 ? s_warp[lane] : Pair{0, 0};
      t = warp_scan(t, lane);
      if (lane < PT_THREADS / 32) s_warp[lane] = t;
    }
    __syncthreads();
    const long long wa = warp ? s_warp[warp - 1].a : 0, wb = warp ? s_warp[warp - 1].b : 0;
    if (i < B) {  // a sum past 32 bits is refused below: its truncated value is never used
      s_cu[i] = (int)(n_sum + wa + w.a - v.a);
      s_base[i] = (int)(p_sum + wb + w.b - v.b);
    }
    n_sum += s_warp[PT_THREADS / 32 - 1].a;
    p_sum += s_warp[PT_THREADS / 32 - 1].b;
    __syncthreads();
  }
  int err = s_err;
  if (n_sum > cap) err |= PT_SLOTS;
  if (p_sum > n_free) err |= PT_POOL;
  const int N = err ? 0 : (int)n_sum, need = err ? 0 : (int)p_sum;
  const int at = blockIdx.x * PT_THREADS + tid, step = gridDim.x * PT_THREADS;
  for (int i = at; i < B; i += step) {
    cu[i] = err ? 0 : s_cu[i];
    total[i] = s_cached[i] + (err ? 0 : fresh[i]);
  }
  if (at == 0) {
    cu[B] = N;
    used[0] = need;
    used[1] = err;
  }
  for (int e = at; e < need; e += step) {
    const int i = last_le(s_base, B, e);
    tables[i * ld + ((s_cached[i] + P - 1) >> shift) + (e - s_base[i])] = free_pages[e];
  }
  for (int t = at; t < cap; t += step) {
    int slot = -1, pos = 0;
    if (t < N) {
      const int i = last_le(s_cu, B, t);
      const int c = s_cached[i], x = c + (t - s_cu[i]);
      const int have = (c + P - 1) >> shift, k = x >> shift;
      // a page taken by this call is read from the free list: its table entry may still be on its way
      const int page = k < have ? tables[i * ld + k] : free_pages[s_base[i] + (k - have)];
      // (a page id that is none gets the largest slot, which lies outside every cache: the append reports it)
      slot = (unsigned)page > 0x7fffffffu >> shift ? 0x7fffffff : (page << shift) + (x & (P - 1));
      pos = x + (start ? start[i] : 0);
    }
    slots[t] = slot;
    positions[t] = pos;
  }
}

// ───────────────────────── append ─────────────────────────
// Row t of qkv = [q heads | k heads | v heads] (the QKV GEMM's output): q' = rot(q + b; pos), K row = rot(k + b;
// pos), V row = v + b, rotate-half pairs (i, i + d/2): (x c - y s, x s + y c) in fp32, rounded once to bf16.
// Bound: HBM (each element read once and written once). A thread owns one item - 8 rotation pairs or 8 V
// elements - of TOK tokens: their rows are fetched before the slots and positions are known, all at once, and the
// item's bias stays in registers. Measured on the GPU: 2.2 us for one token of 64 requests; 61 us for eight prompts of
// 2048 tokens with 40 heads on 8 of 128 (329 MB: 5.4 TB/s, 0.82 of a plain copy's rate).
__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = unpack_bf16(w[k]);
    v[2 * k] = f.x;
    v[2 * k + 1] = f.y;
  }
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  uint4 u;
  u.x = pack_bf16(v[0], v[1]);
  u.y = pack_bf16(v[2], v[3]);
  u.z = pack_bf16(v[4], v[5]);
  u.w = pack_bf16(v[6], v[7]);
  *reinterpret_cast<uint4*>(p) = u;
}
__device__ __forceinline__ void load8f(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

template <int TOK>
__global__ void __launch_bounds__(256, 4)
kv_append_kernel(const __nv_bfloat16* __restrict__ qkv, long long ld, const float* __restrict__ bias,
                 const float* __restrict__ cosT, const float* __restrict__ sinT, int max_pos,
                 const int* __restrict__ slots, const int* __restrict__ positions, __nv_bfloat16* __restrict__ q,
                 __nv_bfloat16* __restrict__ kc, __nv_bfloat16* __restrict__ vc, int T, int nh, int nkv, int d,
                 int shift, int num_pages) {
  const int half = d / 2, gph = half / 8;  // rotation groups per head
  const int rot = (nh + nkv) * gph, items = rot + nkv * d / 8;
  const int j = blockIdx.y * blockDim.x + threadIdx.x;
  if (j >= items) return;
  const bool rotated = j < rot;
  const int head = rotated ? j / gph : (j - rot) / (d / 8) + nh + nkv;
  const int i0 = rotated ? (j - head * gph) * 8 : (j - rot) % (d / 8) * 8;
  const int c0 = head * d + i0, t0 = blockIdx.x * TOK, P = 1 << shift;
  uint4 ra[TOK], rb[TOK];
  int slot[TOK], pos[TOK];
#pragma unroll
  for (int k = 0; k < TOK; ++k) {
    slot[k] = -1;
    if (t0 + k < T) {
      const __nv_bfloat16* src = qkv + (t0 + k) * ld + c0;
      ra[k] = *reinterpret_cast<const uint4*>(src);
      if (rotated) rb[k] = *reinterpret_cast<const uint4*>(src + half);
      slot[k] = slots[t0 + k];
      pos[k] = positions[t0 + k];
    }
  }
  float b0[8] = {}, b1[8] = {};
  if (bias) {
    load8f(bias + c0, b0);
    if (rotated) load8f(bias + c0 + half, b1);
  }
#pragma unroll
  for (int k = 0; k < TOK; ++k) {
    const int page = slot[k] >> shift;
    if (slot[k] < 0) continue;
    if (page >= num_pages || pos[k] < 0 || pos[k] >= max_pos) {
      dt_report(DT_ERR_BOUNDS, 700);
      continue;
    }
    __nv_bfloat16* dst;
    if (head < nh) {
      dst = q + (long long)(t0 + k) * nh * d + c0;
    } else {
      const int h = rotated ? head - nh : head - nh - nkv;
      dst = (rotated ? kc : vc) + (((long long)page * nkv + h) * P + (slot[k] & (P - 1))) * d + i0;
    }
    float a[8];
    unpack8(ra[k], a);
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] += b0[i];
    if (rotated) {
      float b[8], c[8], s[8], o[8];
      unpack8(rb[k], b);
      load8f(cosT + (long long)pos[k] * half + i0, c);
      load8f(sinT + (long long)pos[k] * half + i0, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        b[i] += b1[i];
        o[i] = a[i] * c[i] - b[i] * s[i];
        b[i] = a[i] * s[i] + b[i] * c[i];
      }
      store8(dst, o);
      store8(dst + half, b);
    } else {
      store8(dst, a);
    }
  }
}

}  // namespace

// Arguments travel in one struct (pointers and 64-bit values first, then ints, no padding): a caller through a
// foreign-function interface packs it in one go, and the small calls here are bound by what a call costs.
// page_size = 1 << shift. `tables` rows are `ld` ints apart, `width` of them usable.
struct PageTablesArgs {
  const int *cached, *fresh, *start, *free_pages;
  int *tables, *slots, *positions, *cu, *total, *used;
  long long ld;
  int n_free, width, cap, B, shift, reserved;
};
// The kernel may take more than 48 KB of shared memory (its static part counts too, hence the KB less) once this has
// been asked of the device; one limit for every call, so that no thread lowers another's.
static int page_tables_prepared(int smem) {
  constexpr int MAX_DEVICES = 64;
  static std::atomic<bool> done[MAX_DEVICES];
  if (smem <= 47 * 1024) return 0;
  int dev = 0;
  DT_CUDA_RET(cudaGetDevice(&dev));
  if (dev >= MAX_DEVICES) return -12;
  if (done[dev].load(std::memory_order_acquire)) return 0;
  DT_CUDA_RET(cudaFuncSetAttribute(page_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   3 * PT_MAX_REQUESTS * (int)sizeof(int)));
  done[dev].store(true, std::memory_order_release);
  return 0;
}
DT_API int dt_page_tables(const PageTablesArgs* args, cudaStream_t st) {
  const PageTablesArgs& a = *args;
  if (a.B < 1 || a.B > PT_MAX_REQUESTS || a.cap < 0 || a.n_free < 0 || a.width < 0 || a.shift < 0 || a.shift > 16)
    return -10;
  const long long B = a.B, cap = a.cap;
  const Span out[] = {span_rows(a.tables, B, 4LL * a.width, 4 * a.ld), span(a.slots, 4 * cap), span(a.positions, 4 * cap),
                      span(a.cu, 4 * (B + 1)), span(a.total, 4 * B), span(a.used, 8)};
  const Span in[] = {span(a.cached, 4 * B), span(a.fresh, 4 * B), span(a.start, 4 * B), span(a.free_pages, 4LL * a.n_free)};
  if (outputs_shared(out, in)) return -13;
  const int smem = 3 * a.B * (int)sizeof(int);
  const int rc = page_tables_prepared(smem);
  if (rc) return rc;
  const int work = a.cap > a.B ? a.cap : a.B;
  int grid = (work + 2 * PT_THREADS - 1) / (2 * PT_THREADS);
  if (grid > 148) grid = 148;
  page_tables_kernel<<<grid, PT_THREADS, smem, st>>>(a.cached, a.fresh, a.start, a.free_pages, a.n_free, a.tables, a.ld,
                                                     a.width, a.slots, a.positions, a.cap, a.cu, a.total, a.used, a.B,
                                                     a.shift);
  return (int)cudaGetLastError();
}

// Whether two sets of rows share memory (spans.h): 0 or 1.
DT_API int dt_spans_meet(const void* p, long long rows, long long bytes, long long stride, const void* p2, long long rows2,
                         long long bytes2, long long stride2) {
  return spans_meet(span_rows(p, rows, bytes, stride), span_rows(p2, rows2, bytes2, stride2));
}

struct KvAppendArgs {
  const void* qkv;
  const float *bias, *cosT, *sinT;
  const int *slots, *positions;
  void *q, *kc, *vc;
  long long ld;
  int max_pos, T, nh, nkv, d, shift, num_pages, reserved;
};
DT_API int dt_kv_append(const KvAppendArgs* args, cudaStream_t st) {
  const KvAppendArgs& a = *args;
  const int T = a.T, nh = a.nh, nkv = a.nkv, d = a.d;
  if (T < 0 || nh < 1 || nkv < 1 || d < 16 || d % 16 || a.ld % 8 || a.shift < 0 || a.shift > 16 || a.num_pages < 1)
    return -10;
  if ((reinterpret_cast<uintptr_t>(a.qkv) | reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.kc) |
       reinterpret_cast<uintptr_t>(a.vc) | reinterpret_cast<uintptr_t>(a.bias) | reinterpret_cast<uintptr_t>(a.cosT) |
       reinterpret_cast<uintptr_t>(a.sinT)) & 15)
    return -11;
  if (T == 0) return 0;
  const long long cache = 2LL * a.num_pages * nkv * d << a.shift, W = (long long)(nh + 2 * nkv) * d;
  const Span out[] = {span(a.q, 2LL * T * nh * d), span(a.kc, cache), span(a.vc, cache)};
  const Span in[] = {span_rows(a.qkv, T, 2 * W, 2 * a.ld), span(a.bias, 4 * W), span(a.cosT, 2LL * a.max_pos * d),
                     span(a.sinT, 2LL * a.max_pos * d), span(a.slots, 4LL * T), span(a.positions, 4LL * T)};
  if (outputs_shared(out, in)) return -13;
  const int items = (nh + nkv) * (d / 16) + nkv * d / 8;
  const int threads = items >= 256 ? 256 : (items + 31) / 32 * 32;
  const bool wide = T >= 2048;  // enough tokens that half of the blocks still fills the GPU
  const dim3 grid(wide ? (T + 1) / 2 : T, (items + threads - 1) / threads);
  (wide ? kv_append_kernel<2> : kv_append_kernel<1>)<<<grid, threads, 0, st>>>(
      reinterpret_cast<const __nv_bfloat16*>(a.qkv), a.ld, a.bias, a.cosT, a.sinT, a.max_pos, a.slots, a.positions,
      reinterpret_cast<__nv_bfloat16*>(a.q), reinterpret_cast<__nv_bfloat16*>(a.kc),
      reinterpret_cast<__nv_bfloat16*>(a.vc), T, nh, nkv, d, a.shift, a.num_pages);
  return (int)cudaGetLastError();
}
