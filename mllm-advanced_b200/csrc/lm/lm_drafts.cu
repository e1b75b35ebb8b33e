// Logits to probabilities, and drafted tokens against the target's probabilities (include/mllmb200_lm.h).  Both work a row
// of the vocabulary at a time: a cluster of CTAs per row, each holding its part in shared memory or registers, so that the
// row is read once; what the parts have to tell one another goes through distributed shared memory.
#include <cmath>

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

// ------------------------------------------------------------------------------------------ probabilities
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
  if (ctas > 1) cluster_sync_all();
  else __syncthreads();
  for (int r = 0; r < ctas; ++r) {
    better(mx, at, ctas > 1 ? ld_remote(&s_max, r) : s_max, ctas > 1 ? ld_remote(&s_first, r) : s_first);
    odd = odd || (ctas > 1 ? ld_remote(&s_sum, r) : s_sum) != 0.0f;
  }
  if (ctas > 1) cluster_sync_all();
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
  if (ctas > 1) cluster_sync_all();
  else __syncthreads();
  sum = 0.0f;
  for (int r = 0; r < ctas; ++r) sum += ctas > 1 ? ld_remote(&s_sum, r) : s_sum;
  if (ctas > 1) cluster_sync_all();
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

// grid (cluster, sequences)
__global__ void __launch_bounds__(kDrThreads) lm_verify_kernel(VerifyArgs a) {
  __shared__ double s_rest[kDrWarps], s_all[kDrWarps], s_sum[2], s_scan[kDrWarps];
  __shared__ int s_n, s_kind, s_found, s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, ctas = gridDim.x, part = blockIdx.x, seq = blockIdx.y, k = a.drafts;
  pdl_launch_dependents();
  pdl_wait_prior();
  const float* target = a.target + seq * a.t_seq;
  const float* draft = a.draft + seq * a.d_seq;
  const int* tokens = a.tokens + seq * a.ld_tokens;
  if (warp == 0) {  // first place that is refused (kind 1) or without a drafted token (kind 0)
    int n = k, kind = 0;
    for (int i0 = 0; i0 < k; i0 += 32) {
      const int i = i0 + lane;
      bool ends = false, refused = false;
      if (i < k) {
        const int x = tokens[i];
        ends = x < 0 || x >= a.vocab;
        if (!ends) {
          const double p = mass_of(target[i * a.t_row + x]), q = mass_of(draft[i * a.d_row + x]);
          refused = !((double)a.accept[seq * a.ld_accept + i] * q < p);
        }
      }
      const unsigned hit = __ballot_sync(0xffffffffu, ends || refused);
      if (hit) {
        const int who = __ffs(hit) - 1;
        n = i0 + who;
        kind = __shfl_sync(0xffffffffu, (int)refused, who);
        break;
      }
    }
    if (lane == 0) s_n = n, s_kind = kind;
  }
  __syncthreads();
  const int n = s_n;
  const bool refused = s_kind;
  const float* p = target + n * a.t_row;
  const float* q = draft + (refused ? n * a.d_row : 0);
  const int per = ((a.vocab + ctas - 1) / ctas + 3) / 4 * 4, v0 = min(part * per, a.vocab), v1 = min(v0 + per, a.vocab);
  // a thread's share: consecutive numbers
  const int each = (v1 - v0 + kDrThreads - 1) / kDrThreads, t0 = min(v0 + tid * each, v1), t1 = min(t0 + each, v1);
  double rest = 0.0, all = 0.0;
  for (int i = t0; i < t1; ++i) {
    const double x = mass_of(p[i]);
    all += x;
    if (refused) rest += fmax(x - mass_of(q[i]), 0.0);
  }
  auto warp_sum = [](double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  const double wr = warp_sum(rest), wa = warp_sum(all);
  if (lane == 0) s_rest[warp] = wr, s_all[warp] = wa;
  __syncthreads();
  if (tid == 0) {
    double r = 0.0, l = 0.0;
    for (int w = 0; w < kDrWarps; ++w) r += s_rest[w], l += s_all[w];
    s_sum[0] = r, s_sum[1] = l;
    s_found = 0x7fffffff, s_last = -1;
  }
  cluster_sync_all();
  double total_rest = 0.0, total_all = 0.0, before[2] = {0.0, 0.0};
  for (int r = 0; r < ctas; ++r) {
    const double x = ld_remote(&s_sum[0], r), y = ld_remote(&s_sum[1], r);
    if (r < part) before[0] += x, before[1] += y;
    total_rest += x, total_all += y;
  }
  const bool from_rest = refused && total_rest > 0.0;
  const double total = from_rest ? total_rest : total_all, goal = mass_of(a.pick[seq]) * total;
  // running sums of the threads
  double up = from_rest ? rest : all;
  const double own = up;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double v = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += v;
  }
  if (lane == 31) s_scan[warp] = up;
  __syncthreads();
  double run = before[from_rest ? 0 : 1] + (up - own);
  for (int w = 0; w < warp; ++w) run += s_scan[w];
  int found = 0x7fffffff, last = -1;
  for (int i = t0; i < t1; ++i) {
    double x = mass_of(p[i]);
    if (from_rest) x = fmax(x - mass_of(q[i]), 0.0);
    run += x;
    if (x > 0.0) last = i;
    if (x > 0.0 && run > goal && i < found) found = i;
  }
  if (found != 0x7fffffff) atomicMin(&s_found, found);
  if (last >= 0) atomicMax(&s_last, last);
  cluster_sync_all();
  if (part == 0 && tid == 0) {
    for (int r = 0; r < ctas; ++r) {
      found = min(found, ld_remote(&s_found, r));
      last = max(last, ld_remote(&s_last, r));
    }
    int* out = a.out + seq * a.ld_out;
    for (int i = 0; i <= k; ++i) out[i] = i < n ? tokens[i] : i == n ? (found != 0x7fffffff ? found : last) : -1;
    a.accepted[seq] = n;
  }
  cluster_sync_all();
}

int cluster_for(int rows, int vocab) {
  int c = 1;
  while (c < 8 && rows * c < 2 * kSms && vocab / (2 * c) >= 1024) c *= 2;
  return c;
}

template <class T>
cudaError_t launch_probabilities(const void* logits, long long ld, int rows, int vocab, float t, float* out, long long ld_out, cudaStream_t s) {
  const int c = cluster_for(rows, vocab);
  for (int r0 = 0; r0 < rows; r0 += 65535) {
    const int n = rows - r0 < 65535 ? rows - r0 : 65535;
    const cudaError_t r = launch_pdl_cluster(lm_probabilities_kernel<T>, dim3(c, n), dim3(kDrThreads), dim3(c, 1, 1), 0, s,
                                             static_cast<const T*>(logits) + r0 * ld, ld, vocab, t > 0.0f ? std::fmin(1.0f / t, 3.402823466e+38f) : 0.0f, t == 0.0f, out + r0 * ld_out, ld_out);
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
  if (!seqs) return MLLMB200_OK;
  if (!target || !pick || !accepted || !out || (drafts && (!draft || !tokens || !accept))) return MLLMB200_INVALID_ARG;
  VerifyArgs a{target, draft, accept, pick, tokens, t_seq, t_row, d_seq, d_row, ld_tokens, ld_accept, ld_out, 0, drafts, vocab, accepted, out};
  const int c = cluster_for(seqs, vocab);
  for (int s0 = 0; s0 < seqs; s0 += 65535) {
    VerifyArgs b = a;
    b.seqs = seqs - s0 < 65535 ? seqs - s0 : 65535;
    b.target += s0 * t_seq, b.pick += s0, b.accepted += s0, b.out += s0 * ld_out;
    if (drafts) b.draft += s0 * d_seq, b.tokens += s0 * ld_tokens, b.accept += s0 * ld_accept;
    const cudaError_t r = launch_pdl_cluster(lm_verify_kernel, dim3(c, b.seqs), dim3(kDrThreads), dim3(c, 1, 1), 0, static_cast<cudaStream_t>(stream), b);
    if (r != cudaSuccess) return MLLMB200_CUDA_ERROR;
  }
  return MLLMB200_OK;
}

}  // extern "C"
