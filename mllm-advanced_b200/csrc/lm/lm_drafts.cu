// Logits to probabilities, and drafted tokens against the target's probabilities (include/mllmb200_lm.h).  Both work a row
// of the vocabulary at a time: a cluster of CTAs per row, each holding its part in shared memory or registers, so that the
// row is read once; what the parts have to tell one another goes through distributed shared memory.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "../device_common.cuh"
#include "lm_paged.h"

namespace mllmb200 {
namespace lm {
namespace {

constexpr int kDrThreads = 256, kDrWarps = kDrThreads / 32;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class V>
__device__ __forceinline__ V ld_remote(const V* local, uint32_t rank);
template <>
__device__ __forceinline__ float ld_remote(const float* local, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(local, rank)) : "memory");
  return v;
}
template <>
__device__ __forceinline__ double ld_remote(const double* local, uint32_t rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(map_to_cta(local, rank)) : "memory");
  return v;
}
template <>
__device__ __forceinline__ int ld_remote(const int* local, uint32_t rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(map_to_cta(local, rank)) : "memory");
  return v;
}

// Cluster barriers in the form that wants nothing of the warps: what stands before them here depends on the lane, and the .aligned form is
// only defined where a warp's threads execute it together.
__device__ __forceinline__ void cluster_here() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_here_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_all() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void cluster_meet() {
  cluster_here();
  cluster_all();
}

constexpr int kRowThreads = 512, kRowWarps = kRowThreads / 32, kRowItems = 10;  // a CTA's part of a row: up to 10 x 4 numbers a thread
constexpr int kRowMost = 8 * kRowThreads * 4 * kRowItems;                        // a cluster of 8 CTAs holds rows up to here

// Numbers i .. i + 3 of a row, `fill` before `begin` and from `end` on.  VEC: i is a multiple of 4 and the row lies on 4 numbers; else
// the four are kRowThreads apart.
template <bool VEC, class T>
__device__ __forceinline__ void load4(const T* row, int i, int begin, int end, float fill, float (&v)[4]) {
  if (VEC && i >= begin && i + 3 < end) {
    if constexpr (sizeof(T) == 4) {
      const float4 x = *reinterpret_cast<const float4*>(row + i);
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(row + i);
      const T* t = reinterpret_cast<const T*>(&x);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = to_f32(t[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = i + e * (VEC ? 1 : kRowThreads);
      v[e] = at >= begin && at < end ? to_f32(row[at]) : fill;
    }
  }
}
// The same as bits, -inf outside: numbers of 16 bits are taken apart when all loads are under way (384 rows of 151936 in bf16 otherwise
// wait for one load after the other: 147 us).
template <class T>
__device__ __forceinline__ uint2 bits4(const T* row, int i, int begin, int end) {
  if (i >= begin && i + 3 < end) return *reinterpret_cast<const uint2*>(row + i);
  const uint32_t low = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
  uint32_t b[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) b[e] = i + e >= begin && i + e < end ? reinterpret_cast<const uint16_t*>(row)[i + e] : low;
  return make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
}
// first number of a thread's item k in a part that starts at v0
template <bool VEC>
__device__ __forceinline__ int item_at(int v0, int k, int tid) {
  return VEC ? v0 + (k * kRowThreads + tid) * 4 : v0 + k * kRowThreads * 4 + tid;
}
template <bool VEC>
__device__ __forceinline__ int element(int i, int e) { return VEC ? i + e : i + e * kRowThreads; }

// ------------------------------------------------------------------------------------------ probabilities
// grid (cluster, rows): every CTA reads its part of the row once, all loads in flight, and keeps it in registers.  A thread takes its
// weights against its own maximum; the warps' maxima and sums go to every CTA of the cluster, so that one barrier settles the
// row.  Bound by memory, 8 bytes a number, and by what a CTA does between its loads and its stores (two of them share an SM).
// VEC: rows of logits and of probabilities lie alike in groups of four numbers, a row's first number `sh` places into one.
// AHEAD: grid (cluster, fewer than the rows): a cluster takes every gridDim.y-th row, and copies the next one into shared memory, each
// thread its own numbers, as soon as it has the current one in registers.
// Everything is fp32.  A number passes two exponentials of the special-function unit (2^-22 of the result each), a sum up to four: 1.08e-7 of
// the 2-norm off; with the library's exponential for the numbers 1.06e-7, and 3 % slower.
// 384 rows of 151936, one call after the other: 95 us, 96 with an odd distance of rows, 94 from bf16.  452 with three passes of scalar loads
// over the row, 115 with four barriers and exact exponentials, 105 where all warps send to all CTAs and so wait for their stores
// of the row before, 416 where rows of an odd distance are read number by number.
template <class T, int ITEMS, bool VEC, bool AHEAD>
__global__ void __launch_bounds__(kRowThreads, 2) lm_probability_rows_kernel(const T* __restrict__ logits, long long ld, int rows, int vocab, int per, float inv_t,
                                                                          bool greedy, float* __restrict__ out, long long ld_out) {
  static_assert(VEC || !AHEAD);
  extern __shared__ uint4 s_ahead[];                       // AHEAD: four numbers a thread and item
  __shared__ float2 s_warps[kRowWarps], s_ctas[AHEAD ? 2 : 1][8];  // {maximum, sum or place} of every warp, of every CTA (rows in turn)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, ctas = gridDim.x, part = blockIdx.x;
  cluster_here_relaxed();
  pdl_launch_dependents();
  pdl_wait_prior();
  constexpr int kEach = 4 * sizeof(T);
  const uint32_t place = smem_u32(s_ahead);
  auto shift = [&](const T* z) { return VEC ? (int)(reinterpret_cast<uintptr_t>(z) / sizeof(T) & 3) : 0; };
  auto request = [&](int row, int me) {
    const T* z = logits + row * ld;
    const int sh = shift(z), v1 = min(part * per + per, sh + vocab);
    z -= sh;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int i = item_at<VEC>(part * per, k, me), n = i >= sh && i + 3 < v1 ? kEach : 0;
      const T* from = z + (n ? i : 0);  // (a group of four begins there also where nothing is read)
      if constexpr (kEach == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(place + (k * kRowThreads + me) * kEach), "l"(from), "r"(n) : "memory");
      else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(place + (k * kRowThreads + me) * kEach), "l"(from), "r"(n) : "memory");
    }
    paged_commit();
  };
  if (AHEAD) request(blockIdx.y, tid);
  for (int row = blockIdx.y, turn = 0; row < rows; row += gridDim.y, ++turn) {
    int me = tid;
    asm volatile("" : "+r"(me));  // (places are worked out where they are used: there are no registers to keep them)
    float2* s_pairs = s_ctas[AHEAD ? turn & 1 : 0];
    const T* z = logits + row * ld;
    const int sh = shift(z), v0 = part * per, v1 = min(v0 + per, sh + vocab);  // counted from `sh` numbers before the row
    z -= sh;
    float x[ITEMS][4], mx = -INFINITY;
    if (AHEAD) {
      paged_wait<0>();
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) {
        const int i = item_at<VEC>(v0, k, me);
        if (i >= sh && i + 3 < v1) load4<VEC>(reinterpret_cast<const T*>(s_ahead) + (k * kRowThreads + me) * 4, 0, 0, 4, 0.0f, x[k]);
        else load4<VEC>(z, i, sh, v1, -INFINITY, x[k]);
      }
      if (row + gridDim.y < rows) request(row + gridDim.y, me);
    } else if constexpr (VEC && sizeof(T) == 2) {
      uint2 bits[ITEMS];
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) bits[k] = bits4(z, item_at<VEC>(v0, k, me), sh, v1);
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k][e] = to_f32(reinterpret_cast<const T*>(&bits[k])[e]);
    } else {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) load4<VEC>(z, item_at<VEC>(v0, k, me), sh, v1, -INFINITY, x[k]);
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = fmaxf(mx, x[k][e]);
    const float t2 = fminf(inv_t * kPagedLog2e, 3.402823466e+38f), base = mx > -INFINITY ? mx : 0.0f;
    float top = mx, second = 0.0f;  // of the warp
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (greedy) {
      int at = 0x7fffffff;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (x[k][e] == top) at = min(at, element<VEC>(item_at<VEC>(v0, k, me), e));
      second = __int_as_float((int)__reduce_min_sync(0xffffffffu, (unsigned)at));
    } else {
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[k][e] = paged_exp2((x[k][e] - base) * t2);  // (a NaN, or inf - inf: a NaN, and so the sum, and every probability)
          sum += x[k][e];
        }
      if (sum != 0.0f) sum *= paged_exp2((base - (top > -INFINITY ? top : 0.0f)) * t2);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      second = sum;
    }
    // {maximum, sum or place} of those that lanes have
    auto join = [&](float2 mine) {
      float best = mine.x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
      if (greedy) {
        const unsigned at = mine.x == best && best > -INFINITY ? (unsigned)__float_as_int(mine.y) : 0x7fffffffu;
        return make_float2(best, __int_as_float((int)__reduce_min_sync(0xffffffffu, at)));
      }
      float total = mine.y == 0.0f ? 0.0f : mine.y * paged_exp2((mine.x - (best > -INFINITY ? best : 0.0f)) * t2);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      return make_float2(best, total);
    };
    const float2 none = make_float2(-INFINITY, greedy ? __int_as_float(0x7fffffff) : 0.0f);
    if (lane == 0) s_warps[warp] = make_float2(top, second);
    if (turn == 0) {
      __syncwarp();
      cluster_all();  // every CTA has begun
    }
    __syncthreads();
    if (warp == 0) {
      const float2 ours = join(lane < kRowWarps ? s_warps[lane] : none);
      if (lane < ctas) {
        const uint32_t to = map_to_cta(s_pairs + part, lane);
        st_cluster_f32(to, ours.x);
        st_cluster_f32(to + 4, ours.y);
      }
      __syncwarp();
      cluster_here();
    } else {
      cluster_here_relaxed();  // (with nothing to hand over: it does not wait for the last row's stores)
    }
    cluster_all();
    asm volatile("" : "+r"(me));
    const float2 all = join(lane < ctas ? s_pairs[lane] : none);
    if (greedy) {
      const int at = __float_as_int(all.y);
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k][e] = element<VEC>(item_at<VEC>(v0, k, me), e) == at ? 1.0f : 0.0f;
    } else {
      const float at = all.x > -INFINITY ? all.x : 0.0f, total = all.y;
      // (0: nothing but -inf, in the row or among the thread's)
      const float f = total == 0.0f || (mx == -INFINITY && total == total) ? 0.0f : paged_exp2((base - at) * t2) / total;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k][e] *= f;
    }
    float* y = out + row * ld_out - sh;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int i = item_at<VEC>(v0, k, me);
      if (VEC && i >= sh && i + 3 < v1) {
        *reinterpret_cast<float4*>(y + i) = make_float4(x[k][0], x[k][1], x[k][2], x[k][3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (element<VEC>(i, e) >= sh && element<VEC>(i, e) < v1) y[element<VEC>(i, e)] = x[k][e];
      }
    }
  }
}

// Longer rows: three passes.
// grid (cluster, rows).  TEMP0: one at the first largest.
template <class T>
__global__ void __launch_bounds__(kDrThreads) lm_probabilities_kernel(const T* __restrict__ logits, long long ld, int vocab, float inv_t,
                                                                      bool greedy, float* __restrict__ out, long long ld_out) {
  __shared__ float s_red[kDrWarps], s_max, s_sum;
  __shared__ int s_at[kDrWarps], s_first;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, ctas = gridDim.x, part = blockIdx.x, row = blockIdx.y;
  pdl_launch_dependents();
  pdl_wait_prior();
  const T* z = logits + row * ld;
  float* y = out + row * ld_out;
  const int per = ((vocab + ctas - 1) / ctas + 3) / 4 * 4, v0 = min(part * per, vocab), v1 = min(v0 + per, vocab);
  float mx = -INFINITY;
  int at = 0x7fffffff;
  bool odd = false;  // NaN or +inf
  for (int i = v0 + tid; i < v1; i += kDrThreads) {
    const float x = to_f32(z[i]);
    odd = odd || !(x < INFINITY);
    if (x > mx) mx = x, at = i;
  }
  auto better = [](float& m, int& a, float m2, int a2) {
    if (m2 > m || (m2 == m && a2 < a)) m = m2, a = a2;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(mx, at, __shfl_xor_sync(0xffffffffu, mx, o), __shfl_xor_sync(0xffffffffu, at, o));
  if (lane == 0) s_red[warp] = mx, s_at[warp] = at;
  odd = __syncthreads_or(odd);
  for (int w = 0; w < kDrWarps; ++w) better(mx, at, s_red[w], s_at[w]);
  if (tid == 0) s_max = mx, s_first = at, s_sum = odd ? 1.0f : 0.0f;
  if (ctas > 1) cluster_meet();
  else __syncthreads();
  for (int r = 0; r < ctas; ++r) {
    better(mx, at, ctas > 1 ? ld_remote(&s_max, r) : s_max, ctas > 1 ? ld_remote(&s_first, r) : s_first);
    odd = odd || (ctas > 1 ? ld_remote(&s_sum, r) : s_sum) != 0.0f;
  }
  if (ctas > 1) cluster_meet();
  else __syncthreads();
  if (greedy) {
    for (int i = v0 + tid; i < v1; i += kDrThreads) y[i] = i == at ? 1.0f : 0.0f;
    return;
  }
  float sum = 0.0f;
  if (mx > -INFINITY)
    for (int i = v0 + tid; i < v1; i += kDrThreads) sum += expf((to_f32(z[i]) - mx) * inv_t);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_red[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0.0f;
    for (int w = 0; w < kDrWarps; ++w) sum += s_red[w];
    s_sum = sum;
  }
  if (ctas > 1) cluster_meet();
  else __syncthreads();
  sum = 0.0f;
  for (int r = 0; r < ctas; ++r) sum += ctas > 1 ? ld_remote(&s_sum, r) : s_sum;
  if (ctas > 1) cluster_meet();
  for (int i = v0 + tid; i < v1; i += kDrThreads)
    y[i] = odd ? __int_as_float(0x7fffffff) : mx > -INFINITY ? expf((to_f32(z[i]) - mx) * inv_t) / sum : 0.0f;
}

// ------------------------------------------------------------------------------------------ verification
struct VerifyArgs {
  const float *target, *draft, *accept, *pick;
  const int* tokens;
  long long t_seq, t_row, d_seq, d_row, ld_tokens, ld_accept, ld_out;
  int seqs, drafts, vocab;
  int *accepted, *out;
};
__device__ __forceinline__ double mass_of(float p) { return p > 0.0f ? (double)p : 0.0; }

// First place of a sequence that is refused (.y 1) or has no drafted token (.y 0); one warp.
__device__ __forceinline__ int2 first_refused(const VerifyArgs& a, int seq, int lane) {
  const float* target = a.target + seq * a.t_seq;
  const float* draft = a.draft + seq * a.d_seq;
  const int* tokens = a.tokens + seq * a.ld_tokens;
  for (int i0 = 0; i0 < a.drafts; i0 += 32) {
    const int i = i0 + lane;
    bool ends = false, refused = false;
    if (i < a.drafts) {
      const float u = a.accept[seq * a.ld_accept + i];
      const int x = tokens[i];
      ends = x < 0 || x >= a.vocab;
      if (!ends) refused = !((double)u * mass_of(draft[i * a.d_row + x]) < mass_of(target[i * a.t_row + x]));
    }
    const unsigned hit = __ballot_sync(0xffffffffu, ends || refused);
    if (hit) {
      const int who = __ffs(hit) - 1;
      return make_int2(i0 + who, __shfl_sync(0xffffffffu, (int)refused, who));
    }
  }
  return make_int2(a.drafts, 0);
}

// grid (cluster, sequences): one pass over the row (or the two rows) of the first refused place leaves a sum in 64 bits per 128
// numbers in shared memory; these settle on which CTA and which 128 numbers the draw falls, and one warp reads those again.
// What bounds it: latency for a few sequences (tokens, their probabilities, the rows, one after the other), memory for many.
// 64 sequences of 151936 tokens: 19-22 us (61 MB read); 66 where every thread read consecutive numbers, twice.  Rows of an odd distance,
// which target and draft do not share, are read number by number: 45 from cold caches, 29 by four.
template <bool VEC>
__global__ void __launch_bounds__(kRowThreads, 2) lm_verify_kernel(VerifyArgs a, int per) {
  extern __shared__ double s_part[];  // in the order of the row
  __shared__ double s_sum, s_before;
  __shared__ int s_which, s_place[2];
  constexpr int kItem = kRowThreads * 4, kSums = VEC ? kRowWarps : 4 * kRowWarps;  // numbers and sums of a turn
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, ctas = gridDim.x, part = blockIdx.x, seq = blockIdx.y, k = a.drafts;
  pdl_launch_dependents();
  pdl_wait_prior();
  if (warp == 0) {
    const int2 f = first_refused(a, seq, lane);
    if (lane == 0) s_place[0] = f.x, s_place[1] = f.y;
  }
  const double pick = mass_of(a.pick[seq]);
  __syncthreads();
  const int n = s_place[0];
  bool rest = s_place[1];
  const float* p = a.target + seq * a.t_seq + n * a.t_row;
  const float* q = a.draft + seq * a.d_seq + (rest ? n * a.d_row : 0);
  const int v0 = min(part * per, a.vocab), v1 = min(v0 + per, a.vocab), turns = (v1 - v0 + kItem - 1) / kItem, n_sums = turns * kSums;
  auto warp_sum = [](double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  auto mass = [&](float x, float y) { return rest ? fmax(mass_of(x) - mass_of(y), 0.0) : mass_of(x); };
  double total = 0.0, before = 0.0, own = 0.0;
  while (true) {
    constexpr int kAhead = 4;  // turns requested together
    for (int t0 = 0; t0 < turns; t0 += kAhead) {
      float x[kAhead][4], y[kAhead][4] = {};
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        load4<VEC>(p, item_at<VEC>(v0, t0 + u, tid), 0, v1, 0.0f, x[u]);
        if (rest) load4<VEC>(q, item_at<VEC>(v0, t0 + u, tid), 0, v1, 0.0f, y[u]);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (t0 + u >= turns) break;
        if constexpr (VEC) {
          const double v = warp_sum((mass(x[u][0], y[u][0]) + mass(x[u][1], y[u][1])) + (mass(x[u][2], y[u][2]) + mass(x[u][3], y[u][3])));
          if (lane == 0) s_part[(t0 + u) * kSums + warp] = v;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const double v = warp_sum(mass(x[u][e], y[u][e]));
            if (lane == 0) s_part[(t0 + u) * kSums + e * kRowWarps + warp] = v;
          }
        }
      }
    }
    __syncthreads();
    if (warp == 0) {
      double v = 0.0;
      for (int i = lane; i < n_sums; i += 32) v += s_part[i];
      v = warp_sum(v);
      if (lane == 0) s_sum = v;
    }
    cluster_meet();
    total = before = 0.0;
    for (int r = 0; r < ctas; ++r) {
      const double v = ld_remote(&s_sum, r);
      if (r == part) before = total, own = v;
      total += v;
    }
    if (total > 0.0 || !rest) break;
    rest = false;  // refused, and nothing is left of the target's numbers: from the target
    cluster_meet();
  }
  const double goal = fmin(pick * total, total);
  // the CTA that the draw falls on (pick of 1 and beyond: the last that has mass)
  bool mine = own > 0.0 && before <= goal && goal < before + own;
  if (total > 0.0 && goal >= total) {
    int last = -1;
    for (int r = 0; r < ctas; ++r)
      if (ld_remote(&s_sum, r) > 0.0) last = r;
    mine = last == part;
  }
  cluster_here();  // this CTA has read the others
  int* out = a.out + seq * a.ld_out;
  if (part == 0) {
    const int* tokens = a.tokens + seq * a.ld_tokens;
    for (int i = tid; i <= k; i += kRowThreads)
      if (i != n || !(total > 0.0)) out[i] = i < n ? tokens[i] : -1;
    if (tid == 0) a.accepted[seq] = n;
  }
  if (mine) {  // (the same for all threads)
    if (warp == 0) {  // which of the sums: running sums of 32 at a time
      int which = -1, last = -1;
      double run = before, at_which = before, at_last = before;
      for (int i0 = 0; i0 < n_sums && which < 0; i0 += 32) {
        const double v = i0 + lane < n_sums ? s_part[i0 + lane] : 0.0;
        double up = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double t = __shfl_up_sync(0xffffffffu, up, o);
          if (lane >= o) up += t;
        }
        const unsigned some = __ballot_sync(0xffffffffu, v > 0.0), over = __ballot_sync(0xffffffffu, v > 0.0 && run + up > goal);
        if (some) {
          last = i0 + 31 - __clz(some);
          at_last = run + __shfl_sync(0xffffffffu, up - v, 31 - __clz(some));
        }
        if (over) {
          which = i0 + __ffs(over) - 1;
          at_which = run + __shfl_sync(0xffffffffu, up - v, __ffs(over) - 1);
        }
        run += __shfl_sync(0xffffffffu, up, 31);
      }
      if (lane == 0) s_which = which < 0 ? last : which, s_before = which < 0 ? at_last : at_which;
    }
    __syncthreads();
    const int which = s_which;
    if (which % kRowWarps == warp) {
      const int i = item_at<VEC>(v0, which / kSums, tid), only = which / kRowWarps % 4;
      float x[4], y[4] = {};
      load4<VEC>(p, i, 0, v1, 0.0f, x);
      if (rest) load4<VEC>(q, i, 0, v1, 0.0f, y);
      double m[4], up = 0.0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        m[e] = VEC || e == only ? mass(x[e], y[e]) : 0.0;
        up += m[e];
      }
      const double whole = up;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += t;
      }
      double run = s_before + (up - whole);
      int found = 0x7fffffff, last = -1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        run += m[e];
        if (m[e] > 0.0) {
          last = element<VEC>(i, e);
          if (run > goal) found = min(found, last);
        }
      }
      found = __reduce_min_sync(0xffffffffu, found);
      last = __reduce_max_sync(0xffffffffu, last);
      if (lane == 0) out[n] = found != 0x7fffffff ? found : last;
    }
  }
  cluster_all();
}

// Cluster and items per thread for rows held in registers: as few CTAs as hold the row, more while they do not fill the GPU.
struct RowPlan {
  int ctas, per, items;
};
RowPlan row_plan(int rows, int vocab) {
  constexpr int item = kRowThreads * 4;
  RowPlan p{1, 0, 0};
  auto size = [&] { p.per = ((vocab + p.ctas - 1) / p.ctas + 3) / 4 * 4, p.items = (p.per + item - 1) / item; };
  size();
  while (p.ctas < 8 && (p.items > kRowItems || (p.items > 1 && (long long)rows * p.ctas * 2 <= 2 * kSms))) p.ctas *= 2, size();
  return p;
}
// f(instance) for 1, 2, 4, 6, 8 or 10 items
template <class F>
cudaError_t with_items(int items, F f) {
  if (items <= 1) return f(std::integral_constant<int, 1>());
  if (items <= 2) return f(std::integral_constant<int, 2>());
  if (items <= 4) return f(std::integral_constant<int, 4>());
  if (items <= 6) return f(std::integral_constant<int, 6>());
  if (items <= 8) return f(std::integral_constant<int, 8>());
  return f(std::integral_constant<int, 10>());
}
bool on(const void* p, size_t bytes, long long stride = 0, long long stride2 = 0) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride % 4 == 0 && stride2 % 4 == 0;
}

// Clusters of `ctas` that a device holds at a time, 0 where that is not known.
template <class T, int ITEMS>
int resident_clusters(int ctas) {
  static std::atomic<int> known[64][4];
  int dev = 0, log = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return 0;
  while (1 << log < ctas) ++log;
  if ((n = known[dev][log].load(std::memory_order_acquire))) return n;
  const auto kernel = lm_probability_rows_kernel<T, ITEMS, true, true>;
  constexpr int smem = ITEMS * kRowThreads * 4 * sizeof(T);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, 148), cfg.blockDim = dim3(kRowThreads), cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  known[dev][log].store(n, std::memory_order_release);
  return n;
}

template <class T>
cudaError_t launch_probabilities(const void* logits, long long ld, int rows, int vocab, float t, float* out, long long ld_out, cudaStream_t s) {
  const float inv_t = t > 0.0f ? std::fmin(1.0f / t, 3.402823466e+38f) : 0.0f;
  const bool vec = ((reinterpret_cast<uintptr_t>(logits) / sizeof(T) ^ reinterpret_cast<uintptr_t>(out) / 4) & 3) == 0 && (rows == 1 || ((ld ^ ld_out) & 3) == 0);
  const int places = vocab + (vec && !on(out, 16, rows == 1 ? 0 : ld_out) ? 3 : 0);  // (a row may begin inside a group of four)
  for (int r0 = 0; r0 < rows; r0 += 65535) {
    const int n = std::min(rows - r0, 65535);
    const T* z = static_cast<const T*>(logits) + r0 * ld;
    float* y = out + r0 * ld_out;
    cudaError_t r;
    if (places <= kRowMost) {
      const RowPlan p = row_plan(n, places);
      r = with_items(p.items, [&](auto items) {
        constexpr int kItems = decltype(items)::value;
        auto go = [&](auto kernel, int clusters, size_t smem) {
          return launch_pdl_cluster(kernel, dim3(p.ctas, clusters), dim3(kRowThreads), dim3(p.ctas, 1, 1), smem, s, z, ld, n, vocab, p.per, inv_t, t == 0.0f, y, ld_out);
        };
        // (2048 rows of 32000: 89 us with the next row copied ahead, 94 without; 4096 of 2048 22 and 33; clusters of 4 and 8 have enough under way:
        // 1024 of 65536 110 and 98, 384 of 151936 109 and 95)
        const int room = vec && p.ctas <= 2 ? resident_clusters<T, kItems>(p.ctas) : 0;
        if (room && n > room) return go(lm_probability_rows_kernel<T, kItems, true, true>, room, kItems * kRowThreads * 4 * sizeof(T));
        return vec ? go(lm_probability_rows_kernel<T, kItems, true, false>, n, 0) : go(lm_probability_rows_kernel<T, kItems, false, false>, n, 0);
      });
    } else {
      r = launch_pdl_cluster(lm_probabilities_kernel<T>, dim3(8, n), dim3(kDrThreads), dim3(8, 1, 1), 0, s, z, ld, vocab, inv_t, t == 0.0f, y, ld_out);
    }
    if (r != cudaSuccess) return r;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_probability_rows(const float* logits, long long ld, int rows, int vocab, float temperature, float* out, long long ld_out, cudaStream_t s) {
  return launch_probabilities<float>(logits, ld, rows, vocab, temperature, out, ld_out, s);
}

}  // namespace lm
}  // namespace mllmb200

using namespace mllmb200;
using namespace mllmb200::lm;

extern "C" {

int mllmb200_lm_probabilities(const void* logits, int dtype, long long ld, int rows, int vocab, float temperature, float* out, long long ld_out,
                              void* stream) {
  if (rows < 0 || vocab < 1 || ld < 0 || ld_out < vocab || !(temperature >= 0.0f) || std::isinf(temperature)) return MLLMB200_INVALID_ARG;
  if (dtype != MLLMB200_LM_F32 && dtype != MLLMB200_LM_BF16 && dtype != MLLMB200_LM_F16) return MLLMB200_UNSUPPORTED;
  if (vocab > 1 << 30) return MLLMB200_UNSUPPORTED;  // (places in a row, and steps beyond them, are counted in 32 bits)
  if (!rows) return MLLMB200_OK;
  if (!logits || !out) return MLLMB200_INVALID_ARG;
  auto s = static_cast<cudaStream_t>(stream);
  const cudaError_t r = dtype == MLLMB200_LM_F32    ? launch_probabilities<float>(logits, ld, rows, vocab, temperature, out, ld_out, s)
                        : dtype == MLLMB200_LM_BF16 ? launch_probabilities<__nv_bfloat16>(logits, ld, rows, vocab, temperature, out, ld_out, s)
                                                    : launch_probabilities<__half>(logits, ld, rows, vocab, temperature, out, ld_out, s);
  return r == cudaSuccess ? MLLMB200_OK : MLLMB200_CUDA_ERROR;
}

int mllmb200_lm_verify(const float* target, long long t_seq, long long t_row, const float* draft, long long d_seq, long long d_row, const int* tokens,
                       long long ld_tokens, const float* accept, long long ld_accept, const float* pick, int seqs, int drafts, int vocab,
                       int* accepted, int* out, long long ld_out, void* stream) {
  if (seqs < 0 || drafts < 0 || vocab < 1 || ld_out < drafts + 1 || t_seq < 0 || t_row < 0 || d_seq < 0 || d_row < 0 || ld_tokens < 0 || ld_accept < 0)
    return MLLMB200_INVALID_ARG;
  if (vocab > 1 << 20) return MLLMB200_UNSUPPORTED;
  if (!seqs) return MLLMB200_OK;
  if (!target || !pick || !accepted || !out || (drafts && (!draft || !tokens || !accept))) return MLLMB200_INVALID_ARG;
  VerifyArgs a{target, draft, accept, pick, tokens, t_seq, t_row, d_seq, d_row, ld_tokens, ld_accept, ld_out, 0, drafts, vocab, accepted, out};
  const bool vec = on(target, 16, t_seq, t_row) && (!drafts || on(draft, 16, d_seq, d_row));
  auto st = static_cast<cudaStream_t>(stream);
  for (int s0 = 0; s0 < seqs; s0 += 65535) {
    VerifyArgs b = a;
    b.seqs = std::min(seqs - s0, 65535);
    b.target += s0 * t_seq, b.pick += s0, b.accepted += s0, b.out += s0 * ld_out;
    if (drafts) b.draft += s0 * d_seq, b.tokens += s0 * ld_tokens, b.accept += s0 * ld_accept;
    int ctas = 1, per;
    size_t smem;
    auto size = [&] {
      per = ((vocab + ctas - 1) / ctas + 3) / 4 * 4;
      smem = (size_t)((per + kRowThreads * 4 - 1) / (kRowThreads * 4)) * kRowWarps * (vec ? 1 : 4) * sizeof(double);
    };
    size();
    while (ctas < 8 && (smem > 40 * 1024 || ((long long)b.seqs * ctas * 2 <= 2 * kSms && vocab > ctas * kRowThreads * 4))) ctas *= 2, size();  // (all at once)
    auto go = [&](auto kernel) { return launch_pdl_cluster(kernel, dim3(ctas, b.seqs), dim3(kRowThreads), dim3(ctas, 1, 1), smem, st, b, per); };
    const cudaError_t r = vec ? go(lm_verify_kernel<true>) : go(lm_verify_kernel<false>);
    if (r != cudaSuccess) return MLLMB200_CUDA_ERROR;
  }
  return MLLMB200_OK;
}

}  // extern "C"
