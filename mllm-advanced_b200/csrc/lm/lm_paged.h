// A key-value cache in pages: what the operators over it share (include/mllmb200_lm.h says what they compute).
#pragma once
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "../device_common.cuh"
#include "lm_state.h"

namespace mllmb200 {
namespace lm {

// The public structures as the kernels use them.
struct Paged {
  const void *k, *v;
  long long k_page, k_head, k_row, v_page, v_head, v_row;
  const int *table, *lengths, *q_start;
  const int* q_count;  // rows of every sequence; nullptr: q_start[s + 1] - q_start[s]
  int pages, page, kv_heads, dim, vdim, ld_table, max_pages, seqs, rows;
  int tokens;          // rows of every sequence where q_start is nullptr
  const void* q;
  void* out;
  long long q_row, q_head, out_row, out_head;
  const float *sink, *bias;
  int heads, group, bias_max, window, keep;
  int exact;           // prompts on tcgen05: weights in two halves of 16 bits
  float scale2;        // scale log2(e): scores are in base 2
  unsigned bad_page = kDevStatusBadPage, timeout = kDevStatusTimeout;  // what this call reports in the status word: the engine's bits, or the operators'
};

constexpr float kPagedLog2e = 1.4426950408889634f;
// A bias or a sink for scores in base 2.  The type's lowest value stays finite: it stands for "as good as unseen", and a row that has nothing
// else shares its weight out evenly.  (-inf and NaN stay what they are.)
__device__ __forceinline__ float in_base2(float x) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x * kPagedLog2e), "f"(fminf(x, -3.402823466e+38f)));
  return y;
}
constexpr int kLongest = 1 << 30;  // positions that a table's row can name, at most

// A sequence's length, cut to what its row of the table can name.
__device__ __forceinline__ int paged_length(const Paged& a, int s) {
  const int n = a.lengths[s], most = a.max_pages * a.page;
  if (n > most) atomicOr(&g_device_status, a.bad_page);
  return max(0, min(n, most));
}
// Page number of a table place, or -1.
__device__ __forceinline__ int paged_page(const Paged& a, int s, int place) {
  int p = place < a.max_pages ? __ldg(a.table + (size_t)s * a.ld_table + place) : -1;
  if (p < 0 || p >= a.pages) {
    atomicOr(&g_device_status, a.bad_page);
    p = -1;
  }
  return p;
}
// First row and number of rows of a sequence, inside [0, rows).
__device__ __forceinline__ int2 paged_rows(const Paged& a, int s) {
  if (!a.q_start) return make_int2(s * a.tokens, a.tokens);
  const int r0 = a.q_start[s], n = a.q_count ? a.q_count[s] : a.q_start[s + 1] - r0;
  if (r0 < 0 || r0 >= a.rows) return make_int2(0, 0);
  return make_int2(r0, max(0, min(n, a.rows - r0)));
}

// What rows at positions [first, last] see of a sequence: keys [0, head) and [lo, last].  Walked in blocks of B keys (B a
// multiple of 16): `front` blocks from 0, the others from block lo / B on.
struct Seen {
  int head, lo, last, front, blocks;
};
template <int B>
__device__ __forceinline__ Seen paged_seen(const Paged& a, int first, int last) {
  Seen v;
  v.last = last;
  v.lo = a.window ? max(0, first - a.window + 1) : 0;
  v.head = a.window ? min(a.keep, v.lo) : 0;
  v.front = min((v.head + B - 1) / B, v.lo / B);
  v.blocks = last < 0 ? 0 : v.front + last / B + 1 - v.lo / B;
  return v;
}
template <int B>
__device__ __forceinline__ int block_key(const Seen& v, int b) {  // first key of block b
  return (b < v.front ? b : v.lo / B + b - v.front) * B;
}
__device__ __forceinline__ bool seen_by_some(const Seen& v, int j) { return j <= v.last && (j >= v.lo || j < v.head); }
__device__ __forceinline__ bool seen_by(const Paged& a, int pos, int j) {
  return j <= pos && (a.window == 0 || j > pos - a.window || j < a.keep);
}
// keys [j0, j1] are all seen by every row at positions [first, last]
__device__ __forceinline__ bool seen_by_all(const Paged& a, int first, int last, int j0, int j1) {
  return j1 <= first && (a.window == 0 || j0 > last - a.window || j1 < a.keep);
}

constexpr int kDecSeqs = 512;  // sequences of a launch
constexpr int kDecCtas = kSms;  // shares of the work, at most

// Attention of a few tokens per sequence.  An item is (sequence, kv head, block of rows); its keys are walked in blocks of B.  The blocks of all
// items, one after the other, are dealt out evenly: share c is [c T / G, (c + 1) T / G).  An item that lies in one share is
// finished there; of the others every share leaves the maximum, the sum and the unnormalized output of its share: in place 2 c + 1 where
// the item begins in it, else in place 2 c.
struct DecodeWork {
  float* part_o;    // [2 G][rows of an item][vdim]
  float2* part_ml;  // [2 G][rows of an item]
  long long* base;  // [seqs + 1] blocks of a kv head and row block before every sequence
  int row_blocks;
  const int* redo;  // nullptr: always; else only if one of the CTAs' numbers is not 0
};
// (for all threads of a CTA) blocks of every sequence summed up, base[0 .. seqs]; lengths: kept there too unless it is nullptr
template <int B, int THREADS, class N>
__device__ __forceinline__ void sum_blocks(const Paged& a, N* base, int* lengths = nullptr) {
  __shared__ N s_warp[THREADS / 32];
  constexpr int kEach = (kDecSeqs + THREADS - 1) / THREADS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, s0 = tid * kEach;
  N sum[kEach], run = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (s0 + i < a.seqs) {
      const int len = paged_length(a, s0 + i);
      if (lengths) lengths[s0 + i] = len;
      run += paged_seen<B>(a, len - a.tokens, len - 1).blocks;
    }
    sum[i] = run;
  }
  N up = run;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N v = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += v;
  }
  if (lane == 31) s_warp[warp] = up;
  __syncthreads();
  up -= run;
  for (int i = 0; i < warp; ++i) up += s_warp[i];
  if (tid == 0) base[0] = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (s0 + i < a.seqs) base[s0 + i + 1] = up + sum[i];
  __syncthreads();
}
// the sequence that block b lies in
__device__ __forceinline__ int sequence_of(const Paged& a, const long long* base, int items, long long b) {
  int s = 0;
  for (int step = kDecSeqs / 2; step; step /= 2)
    if (s + step < a.seqs && base[s + step] * items <= b) s += step;
  return s;
}
__device__ __forceinline__ int owner_of(long long b, long long total, int ctas) { return (int)(((b + 1) * ctas - 1) / total); }

// Numbers of 16 bits on the tensor cores.  Softmax weights are made relative to a reference that their row's maximum may outgrow by 2^kLag, and
// stored times 2^kLift.  bf16 has fp32's exponents: no lift, and a reference that seldom moves.  fp16 ends at 65504 and lies 2^-24 apart below
// 2^-14: of a row with one large weight the others would be lost (their fp32 sum counts them), so the reference stays within 2^3 and weights
// are lifted to 2^15.  What 16 bits leave of a weight in two numbers is then 2^-22 of it or 2^-37 of the reference, whichever is more (bf16:
// 2^-17 of it).
template <class T>
struct Num;
template <>
struct Num<__nv_bfloat16> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
  static constexpr uint32_t kExponent = 0x7f807f80u;
  static constexpr float kLag = 8.0f, kLift = 0.0f;
};
template <>
struct Num<__half> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    const __half2 h = *reinterpret_cast<const __half2*>(&w);
    return __half22float2(h);
  }
  static constexpr uint32_t kExponent = 0x7c007c00u;
  static constexpr float kLag = 3.0f, kLift = 12.0f;
};
// infinity or NaN in either half
template <class T>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
  constexpr uint32_t lo = Num<T>::kExponent & 0xffffu, hi = Num<T>::kExponent & 0xffff0000u;
  return (w & lo) == lo || (w & hi) == hi;
}

__device__ __forceinline__ void paged_ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void paged_ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void paged_copy16(uint32_t dst, const void* src, bool valid) {  // zeros where not valid (src: any address then)
  const int n = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void paged_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void paged_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float paged_exp2(float x) {  // results below 2^-126 are 0; 2^-22 of the result off at most
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Kernel attributes are set once per device.
template <class F>
cudaError_t once_per_device(std::atomic<unsigned long long>* done, F f) {
  int dev = 0;
  cudaError_t r = cudaGetDevice(&dev);
  if (r != cudaSuccess) return r;
  const unsigned long long bit = 1ull << (dev & 63);
  if (dev < 64 && (done->load(std::memory_order_acquire) & bit)) return cudaSuccess;
  r = f();
  if (r == cudaSuccess && dev < 64) done->fetch_or(bit, std::memory_order_release);
  return r;
}

// Checked launches for the engine: sizes and strides as the public calls take them.
size_t paged_decode_bytes(const Paged& a);  // workspace of launch_paged_decode for a.seqs sequences
cudaError_t launch_paged_decode(const Paged& a, bool f16, void* workspace, cudaStream_t s);
size_t paged_prompt_bytes(const Paged& a);
cudaError_t launch_paged_prompt(const Paged& a, bool f16, void* workspace, cudaStream_t s);
// Rows of a decode step of sequences with one token each: where their keys and values go, and the lengths with them.
cudaError_t launch_paged_prep(cudaStream_t s, int n, const int2* row_sp, const int* table, int ld_table, int page, int2* row_page, int* lengths);
// out fp32 [rows][ld_out] (the checks are those of mllmb200_lm_probabilities)
cudaError_t launch_probability_rows(const float* logits, long long ld, int rows, int vocab, float temperature, float* out, long long ld_out, cudaStream_t s);

// The same on tcgen05, one block of rows per 128 / group tokens; false: not these sizes.  flags [CTAs]: 1 where values that only some
// tokens see were not finite, and the call has to be done on mma.sync.
bool paged_decode_tc_takes(const Paged& a);
int paged_decode_tc_rows(const Paged& a);  // rows of an item
bool launch_paged_decode_tc(const Paged& a, bool f16, const DecodeWork& w, int* flags, cudaStream_t s, cudaError_t* launched);
bool launch_paged_prompt_tc(const Paged& a, bool f16, void* workspace, cudaStream_t s, cudaError_t* launched);

}  // namespace lm
}  // namespace mllmb200
