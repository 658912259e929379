// Logits processor: penalties for repeated tokens, sparse biases and a token mask, one pass over [B, V].
//
// Row b, token v, with c = how often v occurs in the row's answer (history[prompt, len)) and seen = v occurs in
// history[0, len):
//   z = x;  seen: z = z > 0 ? z / r : z * r;  z -= f c + p [c > 0];  z += bias;  not allowed: z = -inf
// in fp32 from fp32 or bf16 logits. Bound: HBM (each logit read and written once): 256 rows of 32768 bf16 logits
// move 50 MB. A block owns SLICE tokens of one row: it starts the loads of its logits and lists together, counts its
// part of the history in shared memory (integer atomics: their order does not matter; the history is read once per
// slice, from L2) and writes its logits under the penalties and the mask. The few biased tokens are added on top,
// each by the list entry that happens to mark it first; where ids are named again the sum goes over the list in its
// order, so there is one result. (Counts of long histories are applied to every element: computing only the listed tokens,
// in a second pass of scattered reads and writes, took 44 us at 256 rows with 4096-token histories, this 20.)
// Measured on the GPU: 3.4 us for one row of 32768; 6.1 us for 64 rows of 50257 fp32 logits with biases and masks
// (26 MB, 4.3 TB/s); 20 us for 256 rows of 32768 bf16 logits with histories of 4096, biases and masks (54 MB, 2.7
// TB/s): there 71% of the issue slots are taken, by the history and by the counter of every logit.
#include "common.cuh"
#include "spans.h"

// Arguments of the launcher (pointers and 64-bit values first, then ints, no padding). Null pointers leave their part
// out; `lens` goes with `history`, `bias_lens` with the bias lists.
struct LogitsArgs {
  const void* x;
  float* out;
  const int *history, *prompt_lens, *lens;
  const float *repetition, *presence, *frequency;
  const int* bias_ids;
  const float* bias_vals;
  const int* bias_lens;
  const uint32_t* mask;
  long long ldx, ldo, ldh, ldb, ldm;
  int bf16, B, V, max_history, max_bias, reserved;
};

namespace {

constexpr int LP_THREADS = 512, LP_SLICE = 8192, LP_GROUPS = LP_SLICE / 4 / LP_THREADS;
constexpr int LP_IDS = 8, LP_FRONT = LP_IDS * LP_THREADS;  // history entries loaded up front
// bits of a token's counter; the rest counts the answer's occurrences
constexpr int SEEN = (int)0x80000000;  // in the prompt
constexpr int BIASED = 1 << 30;        // in the bias list
constexpr int COUNT = (1 << 23) - 1;
constexpr int LP_MAX_BIAS = 32 * LP_THREADS;  // `mine` below has 32 bits

template <bool BF16>
__device__ __forceinline__ float load1(const void* x, long long i) {
  return BF16 ? bf16_to_f(reinterpret_cast<const __nv_bfloat16*>(x)[i]) : reinterpret_cast<const float*>(x)[i];
}
// four logits as they lie in memory, and as fp32
template <bool BF16>
struct Raw4;
template <>
struct Raw4<false> { using T = float4; };
template <>
struct Raw4<true> { using T = uint2; };
__device__ __forceinline__ float4 widen(const float4& v) { return v; }
__device__ __forceinline__ float4 widen(const uint2& u) {
  const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y);
  return make_float4(a.x, a.y, b.x, b.y);
}

// HIST: a history is given; MASK: a mask. What is not given costs no instructions (the full form is bound by them: its
// ALU runs at 60 % at 256 rows).
template <bool BF16, bool HIST, bool MASK>
__global__ void __launch_bounds__(LP_THREADS, 3) process_logits_kernel(const LogitsArgs a, int head, int vec) {
  extern __shared__ __align__(16) int sh[];  // [SLICE + 4], only with a history or biases
  __shared__ uint32_t mk[LP_SLICE / 32 + 1];
  const int tid = threadIdx.x;
  const int row = blockIdx.y, v0 = blockIdx.x * LP_SLICE, n = min(LP_SLICE, a.V - v0);
  const long long xi = row * a.ldx + v0, oi = row * a.ldo + v0;
  // groups of four start where both the input and the output row are aligned; `lead` elements come before
  const int lead = vec ? (int)((4 - ((row * (a.ldo & 3) + head) & 3)) & 3) : 0;
  const int groups = vec ? max(n - lead, 0) / 4 : 0;
  // the counters start at element -pad, so those of a group lie in one 16-byte word
  int* cnt = sh + ((4 - lead) & 3);
  using Raw = typename Raw4<BF16>::T;
  Raw g[LP_GROUPS];
#pragma unroll
  for (int k = 0; k < LP_GROUPS; ++k) {
    const int i = tid + k * LP_THREADS;
    if (i < groups)
      g[k] = *reinterpret_cast<const Raw*>(reinterpret_cast<const uint8_t*>(a.x) + (xi + lead + 4 * i) * (BF16 ? 2 : 4));
  }
  // everything else this block reads is requested now too; entries past the row's lengths are loaded with the rest
  // (the buffers have them) and dropped below
  const int* h = a.history + row * a.ldh;
  const int* bi = a.bias_ids + row * a.ldb;
  const float* bv = a.bias_vals + row * a.ldb;
  const bool listed = HIST || a.bias_lens;
  int id[LP_IDS], first_bias = -1;
  int len = 0, prompt = 0, nb = 0;
  float r = 1.f, p = 0.f, f = 0.f;
  uint32_t word = 0;
  if (HIST) {
#pragma unroll
    for (int k = 0; k < LP_IDS; ++k) {
      const int t = tid + k * LP_THREADS;
      id[k] = (t < a.max_history ? h[t] : -1) - v0;
    }
    len = min(max(a.lens[row], 0), a.max_history);
    if (a.prompt_lens) prompt = a.prompt_lens[row];
    if (a.repetition) r = a.repetition[row];
    if (a.presence) p = a.presence[row];
    if (a.frequency) f = a.frequency[row];
  }
  if (a.bias_lens) {
    if (tid < a.max_bias) first_bias = bi[tid];
    nb = min(max(a.bias_lens[row], 0), a.max_bias);
  }
  if (MASK) {
    if (tid < (n + 31) / 32) word = a.mask[row * a.ldm + v0 / 32 + tid];
    if (tid < LP_SLICE / 32) mk[tid] = word;
  }
  if (listed)
    for (int i = tid; i < LP_SLICE / 4 + 1; i += LP_THREADS) reinterpret_cast<int4*>(sh)[i] = make_int4(0, 0, 0, 0);
  if (listed || MASK) __syncthreads();
  auto count = [&](int t, int i) {  // history entry t names token i of the slice
    if (t < len && (unsigned)i < (unsigned)n) {
      if (t < prompt) atomicOr(&cnt[i], SEEN);
      else atomicAdd(&cnt[i], 1);
    }
  };
  if (HIST) {
#pragma unroll
    for (int k = 0; k < LP_IDS; ++k) count(tid + k * LP_THREADS, id[k]);
    for (int t = tid + LP_FRONT; t < len; t += LP_THREADS) count(t, h[t] - v0);
    __syncthreads();
  }
  const float r_inv = 1.f / r;  // (one rounding more than the division, far fewer instructions an element)
  auto value = [&](float z, int c, unsigned allowed) {
    if (HIST) {
      z *= c == 0 ? 1.f : z > 0.f ? r_inv : r;
      const float m = __int_as_float((c & COUNT) | 0x4b000000) - 8388608.f;  // the count, below 2^23
      z -= f * m;
      z -= p * fminf(m, 1.f);
    }
    return !MASK || (allowed & 1u) ? z : -INFINITY;
  };
#pragma unroll
  for (int k = 0; k < LP_GROUPS; ++k) {
    const int gi = tid + k * LP_THREADS;
    if (gi < groups) {
      const int i = lead + 4 * gi;
      const float4 z = widen(g[k]);
      const int4 c = HIST ? *reinterpret_cast<const int4*>(cnt + i) : make_int4(0, 0, 0, 0);
      const unsigned ok = MASK ? __funnelshift_r(mk[i >> 5], mk[(i >> 5) + 1], i & 31) : 0xfu;
      *reinterpret_cast<float4*>(a.out + oi + i) =
          make_float4(value(z.x, c.x, ok), value(z.y, c.y, ok >> 1), value(z.z, c.z, ok >> 2), value(z.w, c.w, ok >> 3));
    }
  }
  // what the groups leave out: everything (no common alignment), or up to three elements at either end
  const int rest = n - 4 * groups;
  for (int k = tid; k < rest; k += LP_THREADS) {
    const int i = k < lead ? k : k + 4 * groups;
    a.out[oi + i] = value(load1<BF16>(a.x, xi + i), HIST ? cnt[i] : 0, MASK ? mk[i >> 5] >> (i & 31) : 1u);
  }
  if (!a.bias_lens) return;
  __syncthreads();  // the rows above are written, the counters read
  unsigned mine = 0;  // bit k: entry tid + k LP_THREADS has marked its token
  int again = 0;      // whether some token of the slice is named twice
  for (int e = tid, k = 0; e < nb; e += LP_THREADS, ++k) {
    const int i = (k ? bi[e] : first_bias) - v0;
    if ((unsigned)i >= (unsigned)n) continue;
    if (atomicOr(&cnt[i], BIASED) & BIASED) again = 1;
    else mine |= 1u << k;
  }
  again = __syncthreads_or(again);
  for (int e = tid, k = 0; e < nb; e += LP_THREADS, ++k) {
    if (!(mine >> k & 1u)) continue;
    const int v = k ? bi[e] : first_bias, i = v - v0;
    if (MASK && !((mk[i >> 5] >> (i & 31)) & 1u)) continue;
    float sum = 0.f;
    if (!again) {
      sum = bv[e];
    } else {
      for (int e2 = 0; e2 < nb; ++e2)
        if (bi[e2] == v) sum += bv[e2];
    }
    a.out[oi + i] += sum;
  }
}

}  // namespace

DT_API int dt_process_logits(const LogitsArgs* args, cudaStream_t st) {
  const LogitsArgs& a = *args;
  if (a.B < 0 || a.V < 1 || a.B > 65535 || a.ldx < 0 || a.ldo < a.V || a.max_bias > LP_MAX_BIAS ||
      a.max_history > COUNT)
    return -10;
  if (a.B == 0) return 0;
  const long long B = a.B, V = a.V, e = a.bf16 ? 2 : 4;
  const bool in_place = a.x == a.out && !a.bf16 && a.ldx == a.ldo;  // each element is read by the thread that writes it
  const Span out[] = {span_rows(a.out, B, 4 * V, 4 * a.ldo)};
  const Span in[] = {span_rows(in_place ? nullptr : a.x, B, e * V, e * a.ldx),
                     span_rows(a.history, B, 4LL * a.max_history, 4 * a.ldh),
                     span(a.prompt_lens, 4 * B), span(a.lens, 4 * B),
                     span(a.repetition, 4 * B), span(a.presence, 4 * B), span(a.frequency, 4 * B),
                     span_rows(a.bias_ids, B, 4LL * a.max_bias, 4 * a.ldb),
                     span_rows(a.bias_vals, B, 4LL * a.max_bias, 4 * a.ldb), span(a.bias_lens, 4 * B),
                     span_rows(a.mask, B, (V + 31) / 32 * 4, 4 * a.ldm)};
  if (outputs_shared(out, in)) return -13;
  // Four elements at a time where row and column offsets keep input and output on the same phase of four: both
  // strides agree modulo 4 and both bases sit on the same element of a group.
  const uintptr_t xb = reinterpret_cast<uintptr_t>(a.x), ob = reinterpret_cast<uintptr_t>(a.out);
  const int head = (int)(ob / 4 % 4), xhead = (int)(a.bf16 ? xb / 2 % 4 : xb / 4 % 4);
  const int vec = head == xhead && (a.ldx & 3) == (a.ldo & 3);
  const dim3 grid((a.V + LP_SLICE - 1) / LP_SLICE, a.B);
  const int smem = a.lens || a.bias_lens ? (LP_SLICE + 4) * 4 : 0;
  const bool h = a.lens != nullptr, m = a.mask != nullptr;
  auto* kernel = a.bf16 ? (h ? (m ? process_logits_kernel<true, true, true> : process_logits_kernel<true, true, false>)
                             : (m ? process_logits_kernel<true, false, true> : process_logits_kernel<true, false, false>))
                        : (h ? (m ? process_logits_kernel<false, true, true> : process_logits_kernel<false, true, false>)
                             : (m ? process_logits_kernel<false, false, true> : process_logits_kernel<false, false, false>));
  kernel<<<grid, LP_THREADS, smem, st>>>(a, head, vec);
  return (int)cudaGetLastError();
}
