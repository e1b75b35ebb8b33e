// Operators over a key-value cache in pages (include/mllmb200_lm.h): storing new rows, attention of a few tokens per
// sequence with the lengths split over the GPU, attention of prompts.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "lm_paged_rows.cuh"

namespace mllmb200 {
cudaError_t read_operator_status(cudaStream_t, int* status);

namespace lm {
namespace {

// ------------------------------------------------------------------------------------------ append
// A thread copies 16 bytes of each of ROWS rows; grid (rows / ROWS, pieces / 128).  The rows are on their way while their places are looked
// up: sequence, length and page depend on one another, those of different rows do not.
template <int ROWS>
__global__ void __launch_bounds__(128) lm_pages_append_kernel(Paged a, const void* k, long long k_row, long long k_head, const void* v,
                                                              long long v_row, long long v_head, uint16_t* pool_k, uint16_t* pool_v) {
  pdl_launch_dependents();
  pdl_wait_prior();
  const int kp = a.dim / 8, vp = a.vdim / 8, i = blockIdx.y * 128 + threadIdx.x, row0 = blockIdx.x * ROWS;
  if (i >= a.kv_heads * (kp + vp)) return;
  const bool key = i < a.kv_heads * kp;
  const int j = key ? i : i - a.kv_heads * kp, g = j / (key ? kp : vp), c = (j - g * (key ? kp : vp)) * 8;
  const uint16_t* from = static_cast<const uint16_t*>(key ? k : v) + g * (key ? k_head : v_head) + c;
  uint16_t* to = (key ? pool_k : pool_v) + g * (key ? a.k_head : a.v_head) + c;
  uint4 x[ROWS];
  int seq[ROWS], pos[ROWS], page[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u)
    if (row0 + u < a.rows) x[u] = *reinterpret_cast<const uint4*>(from + (row0 + u) * (key ? k_row : v_row));
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const int row = min(row0 + u, a.rows - 1);
    int t, n;
    if (!a.q_start) {
      seq[u] = row / a.tokens, t = row - seq[u] * a.tokens, n = a.tokens;
    } else {
      int lo = 0, hi = a.seqs;  // last s with q_start[s] <= row
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.q_start[mid] <= row) lo = mid;
        else hi = mid;
      }
      const int2 r = paged_rows(a, lo);
      seq[u] = lo, t = row - r.x, n = r.y;
    }
    pos[u] = row0 + u < a.rows && t >= 0 && t < n ? t - n : 0;  // (0: behind the last row or the last sequence)
  }
#pragma unroll
  for (int u = 0; u < ROWS; ++u) pos[u] = pos[u] < 0 ? a.lengths[seq[u]] + pos[u] : -1;  // (uncut: beyond the table is no page, and no other row's)
#pragma unroll
  for (int u = 0; u < ROWS; ++u) page[u] = pos[u] >= 0 ? paged_page(a, seq[u], pos[u] / a.page) : -1;
#pragma unroll
  for (int u = 0; u < ROWS; ++u)
    if (page[u] >= 0) *reinterpret_cast<uint4*>(to + page[u] * (key ? a.k_page : a.v_page) + pos[u] % a.page * (key ? a.k_row : a.v_row)) = x[u];
}

// ------------------------------------------------------------------------------------------ decode
template <class T, int DV, int MT, int STAGES, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 1) lm_paged_decode_kernel(Paged a, DecodeWork w) {
  constexpr int kDecWarps = WARPS, kDecThreads = 32 * WARPS, kDecB = 16 * WARPS;
  extern __shared__ __align__(16) uint8_t pd_smem[];
  __shared__ long long s_base[kDecSeqs + 1];
  __shared__ float s_m[kDecWarps][16 * MT], s_l[kDecWarps][16 * MT];
  constexpr int kRows = 16 * MT;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ldk = a.dim + 8, ldv = a.vdim + 8;
  T* sQ = reinterpret_cast<T*>(pd_smem);
  T* ring = sQ + kRows * ldk;                            // [warps][stages][16 keys | 16 values]
  float* sO = reinterpret_cast<float*>(ring);            // [warps][rows][vdim], when a share is used up
  const int stage_elems = 16 * (ldk + ldv);
  T* mine = ring + (size_t)warp * STAGES * stage_elems;
  pdl_launch_dependents();
  pdl_wait_prior();
  if (w.redo) {  // again, and only if some CTA of the kernel before asks for it
    bool asked = false;
    for (int i = tid; i < kDecCtas; i += kDecThreads) asked = asked || w.redo[i] != 0;
    if (!__syncthreads_or(asked)) return;
  }
  sum_blocks<kDecB, kDecThreads>(a, s_base);
  if (blockIdx.x == 0)
    for (int i = tid; i <= a.seqs; i += kDecThreads) w.base[i] = s_base[i];
  const int items = a.kv_heads * w.row_blocks, rows = a.group * a.tokens;  // per sequence; per kv head
  const long long total = s_base[a.seqs] * items;
  const int ctas = (int)min((long long)gridDim.x, total);  // (every one of them has something)
  if ((int)blockIdx.x >= ctas) return;
  long long b = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1) / ctas;
  if (w.redo) {  // whole items, so that nothing is left to join
    auto item_start = [&](long long i) { return s_base[i / items] * items + i % items * (s_base[min((int)(i / items) + 1, a.seqs)] - s_base[i / items]); };
    const long long n = (long long)a.seqs * items;
    b = item_start(n * blockIdx.x / ctas), end = item_start(n * (blockIdx.x + 1) / ctas);
  }
  const int mat = lane >> 3, ml = lane & 7, cr = lane >> 3, cc = lane & 7;
  const uint32_t q_addr = smem_u32(sQ + ((mat & 1) * 8 + ml) * ldk + (mat >> 1) * 8);

  while (b < end) {
    const int s = sequence_of(a, s_base, items, b), len = paged_length(a, s), p_first = len - a.tokens, p_last = len - 1;
    const Seen seen = paged_seen<kDecB>(a, p_first, p_last);
    const long long in_seq = b - s_base[s] * items;
    const int item = (int)(in_seq / seen.blocks), blk0 = (int)(in_seq - (long long)item * seen.blocks);
    const int n_blk = (int)min(end - b, (long long)(seen.blocks - blk0));
    const bool begins = blk0 == 0, whole = begins && n_blk == seen.blocks;
    const int kvh = item / w.row_blocks, r0 = (item - kvh * w.row_blocks) * kRows;
    const int2 q_rows = paged_rows(a, s);
    const T* kb = static_cast<const T*>(a.k) + kvh * a.k_head;
    const T* vb = static_cast<const T*>(a.v) + kvh * a.v_head;

    int pids = -1;  // lane i: page of this warp's slice i of 32
    auto fetch = [&](int it) {
      if (it < n_blk) {
        if ((it & 31) == 0) {
          const int j = block_key<kDecB>(seen, blk0 + it + lane) + warp * 16;
          pids = it + lane < n_blk && j <= seen.last && (j + 15 >= seen.lo || j < seen.head) ? paged_page(a, s, j / a.page) : -1;
        }
        const int page = __shfl_sync(0xffffffffu, pids, it & 31), j = block_key<kDecB>(seen, blk0 + it) + warp * 16, at = j % a.page;
        T* dk = mine + (size_t)(it % STAGES) * stage_elems;
        T* dv = dk + 16 * ldk;
        const T* ks = kb + (page < 0 ? 0 : page * a.k_page + at * a.k_row);
        const T* vs = vb + (page < 0 ? 0 : page * a.v_page + at * a.v_row);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int r = cr + u * 4;
          const bool ok = page >= 0 && seen_by_some(seen, j + r);
          for (int c = cc * 8; c < a.dim; c += 64) paged_copy16(smem_u32(dk + r * ldk + c), ok ? ks + r * a.k_row + c : kb, ok);
          for (int c = cc * 8; c < a.vdim; c += 64) paged_copy16(smem_u32(dv + r * ldv + c), ok ? vs + r * a.v_row + c : vb, ok);
        }
      }
      paged_commit();
    };
#pragma unroll
    for (int it = 0; it < STAGES - 1; ++it) fetch(it);
    for (int i = tid; i < kRows * (a.dim / 8); i += kDecThreads) {
      const int r = i / (a.dim / 8), c = (i - r * (a.dim / 8)) * 8, tok = (r0 + r) / a.group, hg = r0 + r - tok * a.group;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (r0 + r < rows && tok < q_rows.y)
        x = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (q_rows.x + tok) * a.q_row + (kvh * a.group + hg) * a.q_head + c);
      *reinterpret_cast<uint4*>(sQ + r * ldk + c) = x;
    }
    float m[MT][2], l[MT][2], o[MT][DV / 8][4];
    int pos[MT][2];
    const float* bias[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = r0 + t * 16 + (lane >> 2) + i * 8, tok = r / a.group;
        m[t][i] = -INFINITY, l[t][i] = 0.0f;
        pos[t][i] = r < rows ? p_first + tok : -1;
        bias[t][i] = a.bias && r < rows ? a.bias + (size_t)(kvh * a.group + r - tok * a.group) * (a.bias_max + 1) : nullptr;
      }
#pragma unroll
      for (int n = 0; n < DV / 8; ++n) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.0f;
    }
    __syncthreads();
    for (int it = 0; it < n_blk; ++it) {
      fetch(it + STAGES - 1);
      paged_wait<STAGES - 1>();
      __syncwarp();
      const int j0 = block_key<kDecB>(seen, blk0 + it) + warp * 16;
      if (j0 <= seen.last && (j0 + 15 >= seen.lo || j0 < seen.head)) {
        const T* tk = mine + (size_t)(it % STAGES) * stage_elems;
        const uint32_t k_addr = smem_u32(tk + ((mat >> 1) * 8 + ml) * ldk + (mat & 1) * 8);
        const uint32_t v_addr = smem_u32(tk + 16 * ldk + ((mat & 1) * 8 + ml) * ldv + (mat >> 1) * 8);
        float sc[MT][2][4] = {};
#pragma unroll 4
        for (int kk = 0; kk < a.dim; kk += 16) {
          uint32_t kf[4];
          paged_ldsm(kf, k_addr + kk * 2);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            uint32_t qf[4];
            paged_ldsm(qf, q_addr + (t * 16 * ldk + kk) * 2);
            Num<T>::mma(sc[t][0], qf, kf[0], kf[1]);
            Num<T>::mma(sc[t][1], qf, kf[2], kf[3]);
          }
        }
        const bool all = seen_by_all(a, p_first, p_last, j0, j0 + 15);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          float alpha[2];
          if (all) weigh_keys<T, 2, true>(a, sc[t], m[t], l[t], alpha, j0, lane, pos[t], bias[t]);
          else weigh_keys<T, 2, false>(a, sc[t], m[t], l[t], alpha, j0, lane, pos[t], bias[t]);
          if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
            for (int n = 0; n < DV / 8; ++n) o[t][n][0] *= alpha[0], o[t][n][1] *= alpha[0], o[t][n][2] *= alpha[1], o[t][n][3] *= alpha[1];
          }
          uint32_t hi[4], lo[4];
          split_weights<T>(sc[t][0], sc[t][1], hi, lo);
          // (keys that no row sees are zeros; with one token a sequence those are all that are masked)
          if (all || a.tokens == 1) weigh_values<T, DV, false>(a, o[t], hi, lo, v_addr, j0, lane, pos[t], 0, 0);
          else weigh_values<T, DV, true>(a, o[t], hi, lo, v_addr, j0, lane, pos[t], max(0, p_first), p_last);
        }
      }
      __syncwarp();
    }
    paged_wait<0>();
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], 1);
        l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], 2);
      }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = t * 16 + (lane >> 2) + i * 8;
        if ((lane & 3) == 0) s_m[warp][r] = m[t][i] - Num<T>::kLift, s_l[warp][r] = l[t][i];  // (what sums and outputs are relative to)
        float* so = sO + ((size_t)warp * kRows + r) * a.vdim + (lane & 3) * 2;
#pragma unroll
        for (int n = 0; n < DV / 8; ++n)
          if (n * 8 < a.vdim) *reinterpret_cast<float2*>(so + n * 8) = make_float2(o[t][n][2 * i], o[t][n][2 * i + 1]);
      }
    __syncthreads();
    const int slot = 2 * blockIdx.x + begins, n_rows = min(kRows, rows - r0);
    for (int i = tid; i < n_rows * a.vdim; i += kDecThreads) {
      const int r = i / a.vdim, d = i - r * a.vdim, tok = (r0 + r) / a.group, h = kvh * a.group + r0 + r - tok * a.group;
      const float sink = whole && a.sink ? in_base2(a.sink[h]) : -INFINITY;
      float mx = sink;
#pragma unroll
      for (int u = 0; u < kDecWarps; ++u) mx = fmaxf(mx, s_m[u][r]);
      const float base = mx == -INFINITY ? 0.0f : mx;
      float sum = whole && a.sink ? exp2f(sink - base) : 0.0f, v = 0.0f;
#pragma unroll
      for (int u = 0; u < kDecWarps; ++u) {
        const float f = exp2f(s_m[u][r] - base);
        sum = fmaf(f, s_l[u][r], sum);
        v = fmaf(f, sO[(size_t)u * kRows * a.vdim + i], v);
      }
      if (whole) {
        if (tok < q_rows.y) {
          T* out = static_cast<T*>(a.out) + (q_rows.x + tok) * a.out_row + h * a.out_head + d;
          *out = T(p_first + tok < 0 ? 0.0f : v / sum);
        }
      } else {
        w.part_o[((size_t)slot * kRows + r) * a.vdim + d] = v;
        if (d == 0) w.part_ml[(size_t)slot * kRows + r] = make_float2(mx, sum);
      }
    }
    b += n_blk;
    __syncthreads();
  }
}

// grid (items of all sequences, rows of an item x PER / 4): joins the shares of a row of an item that lies in several CTAs, PER warps a row;
// zeros for those without keys.
constexpr int kJoinWarps = 4;
template <class T, int PER>
__global__ void __launch_bounds__(32 * kJoinWarps) lm_paged_join_kernel(Paged a, DecodeWork w, int item_rows) {
  __shared__ float s_v[PER > 1 ? kJoinWarps : 1][256], s_sum[kJoinWarps];
  pdl_launch_dependents();
  const int items = a.kv_heads * w.row_blocks, s = blockIdx.x / items, item = blockIdx.x - s * items, warp = PER > 1 ? threadIdx.x >> 5 : 0, lane = threadIdx.x & 31;
  const int kvh = item / w.row_blocks, r = PER > 1 ? blockIdx.y : blockIdx.y * kJoinWarps + (threadIdx.x >> 5), row = (item - kvh * w.row_blocks) * item_rows + r;
  const int tok = row / a.group, h = kvh * a.group + row - tok * a.group;
  pdl_wait_prior();
  if (r >= item_rows || row >= a.group * a.tokens) return;
  const long long b0 = w.base[s] * items, nb = w.base[s + 1] - w.base[s], first = b0 + item * nb, total = w.base[a.seqs] * items;
  const int ctas = (int)min((long long)kDecCtas, total), c0 = nb ? owner_of(first, total, ctas) : 0, n = nb ? owner_of(first + nb - 1, total, ctas) - c0 + 1 : 0;
  if (n == 1) return;  // finished there
  const int2 q_rows = paged_rows(a, s);
  if (tok >= q_rows.y) return;
  const bool nothing = n == 0 || paged_length(a, s) - a.tokens + tok < 0;
  auto slot = [&](int i) { return (size_t)(2 * (c0 + i) + (i == 0)) * item_rows + r; };
  const float sink = a.sink ? in_base2(a.sink[h]) : -INFINITY;
  float mx = sink;
  for (int i = lane; i < n; i += 32) mx = fmaxf(mx, w.part_ml[slot(i)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float base = mx == -INFINITY ? 0.0f : mx;
  float sum = 0.0f, v[8] = {};  // columns 4 lane .. and 128 + 4 lane ..
  for (int i0 = warp; i0 < n; i0 += 32 * PER) {  // lane l: share i0 + PER l
    float f = 0.0f;
    if (i0 + PER * lane < n) {
      const float2 ml = w.part_ml[slot(i0 + PER * lane)];
      f = exp2f(ml.x - base);
      sum = fmaf(f, ml.y, sum);
    }
    const int here = min(32, (n - i0 + PER - 1) / PER);
#pragma unroll 8
    for (int i = 0; i < here; ++i) {
      const float fi = __shfl_sync(0xffffffffu, f, i);
      const float* part = w.part_o + slot(i0 + PER * i) * a.vdim;
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (c * 128 + lane * 4 < a.vdim) {
          const float4 x = *reinterpret_cast<const float4*>(part + c * 128 + lane * 4);
          v[c * 4] = fmaf(fi, x.x, v[c * 4]), v[c * 4 + 1] = fmaf(fi, x.y, v[c * 4 + 1]);
          v[c * 4 + 2] = fmaf(fi, x.z, v[c * 4 + 2]), v[c * 4 + 3] = fmaf(fi, x.w, v[c * 4 + 3]);
        }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  T* out = static_cast<T*>(a.out) + (q_rows.x + tok) * a.out_row + h * a.out_head;
  if constexpr (PER == 1) {
    const float inv = 1.0f / (sum + exp2f(sink - base));
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (c * 128 + lane * 4 < a.vdim)
        *reinterpret_cast<uint2*>(out + c * 128 + lane * 4) =
            nothing ? make_uint2(0, 0) : make_uint2(Num<T>::pack(v[c * 4] * inv, v[c * 4 + 1] * inv), Num<T>::pack(v[c * 4 + 2] * inv, v[c * 4 + 3] * inv));
  } else {
#pragma unroll
    for (int c = 0; c < 2; ++c) *reinterpret_cast<float4*>(&s_v[warp][c * 128 + lane * 4]) = make_float4(v[c * 4], v[c * 4 + 1], v[c * 4 + 2], v[c * 4 + 3]);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    const float inv = 1.0f / ((s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]) + exp2f(sink - base));
    for (int d = threadIdx.x * 2; d < a.vdim; d += 64 * kJoinWarps) {
      const float x = (s_v[0][d] + s_v[1][d]) + (s_v[2][d] + s_v[3][d]), y = (s_v[0][d + 1] + s_v[1][d + 1]) + (s_v[2][d + 1] + s_v[3][d + 1]);
      *reinterpret_cast<uint32_t*>(out + d) = nothing ? 0u : Num<T>::pack(x * inv, y * inv);
    }
  }
}

// ------------------------------------------------------------------------------------------ prompts, any head size
// grid (tiles, kv heads): 64 rows (token, query head of one kv head).
template <class T, int DV>
__global__ void __launch_bounds__(kPpThreads) lm_paged_prompt_kernel(Paged a) {
  extern __shared__ __align__(16) uint8_t pp_smem[];
  pdl_launch_dependents();
  pdl_wait_prior();
  const int toks = kPpRows / a.group;
  const int2 tile = paged_tile(a, blockIdx.x, toks);
  if (tile.x < 0) return;
  const int2 rows = paged_rows(a, tile.x);
  struct Cta {
    __device__ void sync() const { __syncthreads(); }
    __device__ bool any(bool v) const { return __syncthreads_or(v) != 0; }
  };
  paged_prompt_rows<T, DV>(a, pp_smem, Cta{}, threadIdx.x, tile.x, rows.x + tile.y * toks, min(toks, rows.y - tile.y * toks),
                           paged_length(a, tile.x) - rows.y + tile.y * toks, blockIdx.y);
}

// ------------------------------------------------------------------------------------------ host
constexpr int kPagedSmemMax = 220 * 1024;

int dec_stages(const Paged& a) { return a.dim + a.vdim <= 128 ? 5 : 3; }
int dec_warps(const Paged& a) { return a.vdim <= 128 && a.dim + a.vdim <= 256 ? 8 : 4; }
int dec_rows(const Paged& a) { return a.vdim <= 128 && a.group * a.tokens > 16 ? 32 : 16; }
size_t decode_smem(const Paged& a) {
  const size_t rows = dec_rows(a), ring = (size_t)dec_warps(a) * dec_stages(a) * 16 * (a.dim + a.vdim + 16) * 2;
  return rows * (a.dim + 8) * 2 + std::max(ring, dec_warps(a) * rows * a.vdim * 4);
}
size_t up16(size_t n) { return (n + 15) / 16 * 16; }

cudaError_t configure_prompt() {
  static std::atomic<unsigned long long> done{0};
  return once_per_device(&done, [] {
    cudaError_t r = cudaSuccess;
    auto set = [&](auto f) {
      if (r == cudaSuccess) r = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kPagedSmemMax);
    };
    set(lm_paged_prompt_kernel<__nv_bfloat16, 64>), set(lm_paged_prompt_kernel<__nv_bfloat16, 128>), set(lm_paged_prompt_kernel<__nv_bfloat16, 256>);
    set(lm_paged_prompt_kernel<__half, 64>), set(lm_paged_prompt_kernel<__half, 128>), set(lm_paged_prompt_kernel<__half, 256>);
    return r;
  });
}
// f(kernel) for the instance that serves these sizes
template <class T, int DV, int MT, class F>
auto with_decode_rows(const Paged& a, F f) {
  if (dec_warps(a) == 4) return f(lm_paged_decode_kernel<T, DV, MT, 3, 4>);
  return dec_stages(a) == 5 ? f(lm_paged_decode_kernel<T, DV, MT, 5, 8>) : f(lm_paged_decode_kernel<T, DV, MT, 3, 8>);
}
template <class T, class F>
auto with_decode(const Paged& a, F f) {
  const bool two = dec_rows(a) == 32;
  if (a.vdim <= 64) return two ? with_decode_rows<T, 64, 2>(a, f) : with_decode_rows<T, 64, 1>(a, f);
  if (a.vdim <= 128) return two ? with_decode_rows<T, 128, 2>(a, f) : with_decode_rows<T, 128, 1>(a, f);
  return f(lm_paged_decode_kernel<T, 256, 1, 3, 4>);
}
cudaError_t configure_decode() {
  static std::atomic<unsigned long long> done{0};
  return once_per_device(&done, [] {
    cudaError_t r = cudaSuccess;
    auto set = [&](auto f) {
      if (r == cudaSuccess) r = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kPagedSmemMax);
      return r;
    };
    for (int vdim : {64, 80, 128, 256})  // (reaches every instance)
      for (int dim : {16, 128, 256})
        for (int tokens : {1, 32}) {
          Paged a{};
          a.vdim = vdim, a.dim = dim, a.group = 1, a.tokens = tokens;
          with_decode<__nv_bfloat16>(a, set);
          with_decode<__half>(a, set);
        }
    return r;
  });
}

// Layout of the decode workspace for `seqs` sequences of a launch.
struct DecodeSpace {
  size_t ml, base, flags, bytes;
};
DecodeSpace decode_space(const Paged& a, int seqs) {
  DecodeSpace d;
  const size_t rows = (size_t)2 * kDecCtas * std::max(dec_rows(a), paged_decode_tc_takes(a) ? paged_decode_tc_rows(a) : 0);
  d.ml = up16(rows * a.vdim * 4);
  d.base = d.ml + up16(rows * sizeof(float2));
  d.flags = d.base + up16((size_t)(seqs + 1) * sizeof(long long));
  d.bytes = d.flags + kDecCtas * sizeof(int);
  return d;
}

bool aligned(const void* p, long long a, long long b, long long c = 0) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && a % 8 == 0 && b % 8 == 0 && c % 8 == 0;
}

int check_pages(const mllmb200_lm_pages* p, Paged* a) {
  if (!p || p->seqs < 0 || p->rows < 0) return MLLMB200_INVALID_ARG;
  if (p->dtype != MLLMB200_LM_BF16 && p->dtype != MLLMB200_LM_F16) return MLLMB200_UNSUPPORTED;
  if (p->pages < 1 || p->page < 1 || p->kv_heads < 1 || p->dim < 1 || p->vdim < 1 || p->max_pages < 0 || p->ld_table < 0) return MLLMB200_INVALID_ARG;
  if (p->page % 16 || p->dim % 16 || p->vdim % 16 || p->dim > 256 || p->vdim > 256) return MLLMB200_UNSUPPORTED;
  if ((long long)p->max_pages * p->page > kLongest || p->rows > kLongest) return MLLMB200_UNSUPPORTED;
  if (p->seqs && (!p->k || !p->v || !p->lengths || (!p->table && p->max_pages))) return MLLMB200_INVALID_ARG;
  *a = Paged{};
  a->k_page = p->k_page, a->k_head = p->k_head, a->k_row = p->k_row, a->v_page = p->v_page, a->v_head = p->v_head, a->v_row = p->v_row;
  // (the stride of a dimension of one says nothing)
  if (p->kv_heads == 1) a->k_head = p->k_row, a->v_head = p->v_row;
  if (p->pages == 1) a->k_page = p->k_row, a->v_page = p->v_row;
  if (!aligned(p->k, a->k_page, a->k_head, a->k_row) || !aligned(p->v, a->v_page, a->v_head, a->v_row)) return MLLMB200_INVALID_ARG;
  if (!p->q_start && (p->seqs ? p->rows % p->seqs : p->rows)) return MLLMB200_INVALID_ARG;  // (rows that are nobody's would be left as they are)
  a->k = p->k, a->v = p->v;
  a->table = p->table, a->lengths = p->lengths, a->q_start = p->q_start;
  a->pages = p->pages, a->page = p->page, a->kv_heads = p->kv_heads, a->dim = p->dim, a->vdim = p->vdim;
  a->ld_table = p->ld_table, a->max_pages = p->max_pages, a->seqs = p->seqs, a->rows = p->rows;
  a->tokens = p->q_start || !p->seqs ? 0 : p->rows / p->seqs;
  a->bad_page <<= kDevStatusOfOperators, a->timeout <<= kDevStatusOfOperators;
  return MLLMB200_OK;
}
int check_look(const mllmb200_lm_pages* p, const mllmb200_lm_look* l, Paged* a) {
  const int st = check_pages(p, a);
  if (st != MLLMB200_OK) return st;
  if (!l || l->heads < 1 || l->heads % a->kv_heads || l->window < 0 || l->keep < 0 || !(std::fabs(l->scale) <= 3.402823466e+38f)) return MLLMB200_INVALID_ARG;
  if (l->heads / a->kv_heads > 64) return MLLMB200_UNSUPPORTED;
  if (l->bias && l->bias_max < 0) return MLLMB200_INVALID_ARG;
  if (a->rows && (!l->q || !l->out)) return MLLMB200_INVALID_ARG;
  a->q = l->q, a->out = l->out;
  a->q_row = l->q_row, a->q_head = l->q_head, a->out_row = l->out_row, a->out_head = l->out_head;
  if (l->heads == 1) a->q_head = a->dim, a->out_head = a->vdim;
  if (a->rows == 1) a->q_row = (long long)l->heads * a->dim, a->out_row = (long long)l->heads * a->vdim;
  if (!aligned(l->q, a->q_row, a->q_head) || !aligned(l->out, a->out_row, a->out_head)) return MLLMB200_INVALID_ARG;
  a->sink = l->sink, a->bias = l->bias;
  a->heads = l->heads, a->group = l->heads / a->kv_heads, a->bias_max = l->bias_max;
  a->window = std::min(l->window, kLongest), a->keep = std::min(l->keep, kLongest);  // (no position is beyond; differences stay in 32 bits)
  a->scale2 = l->scale * kPagedLog2e;
  a->exact = l->exact != 0;
  return MLLMB200_OK;
}
int check_decode(const mllmb200_lm_pages* p, const mllmb200_lm_look* l, Paged* a) {
  const int st = check_look(p, l, a);
  if (st != MLLMB200_OK) return st;
  if (a->q_start) return MLLMB200_INVALID_ARG;
  return a->tokens > 16 ? MLLMB200_UNSUPPORTED : MLLMB200_OK;
}

// An item lies in kDecCtas / items CTAs or one more.  One warp a row where that is few (five tokens of 32 sequences with 4 key heads: the
// whole call 132 us, with four warps 139), four where it is many (one token of one sequence of 60000, 2 key heads: 34.5 and 22.0).
template <class T>
cudaError_t join_decode(const Paged& a, const DecodeWork& w, int item_rows, cudaStream_t s) {
  const int rows = std::min(item_rows, a.group * a.tokens), items = a.seqs * a.kv_heads * w.row_blocks;
  return items * 8 < kDecCtas ? launch_pdl(lm_paged_join_kernel<T, kJoinWarps>, dim3(items, rows), dim3(32 * kJoinWarps), 0, s, a, w, item_rows)
                              : launch_pdl(lm_paged_join_kernel<T, 1>, dim3(items, (rows + kJoinWarps - 1) / kJoinWarps), dim3(32 * kJoinWarps), 0, s, a, w, item_rows);
}
template <class T>
cudaError_t launch_decode(Paged a, uint8_t* ws, cudaStream_t s) {
  const int all = a.seqs, item_rows = dec_rows(a);
  const DecodeSpace d = decode_space(a, std::min(all, kDecSeqs));
  const size_t smem = decode_smem(a);
  for (int s0 = 0; s0 < all; s0 += kDecSeqs) {
    Paged b = a;
    b.seqs = std::min(kDecSeqs, all - s0);
    b.lengths += s0;
    b.table += (size_t)s0 * a.ld_table;
    if (b.q_start) b.q_start += s0, b.q_count += s0;
    else b.q = static_cast<const T*>(a.q) + (long long)s0 * a.tokens * a.q_row, b.out = static_cast<T*>(a.out) + (long long)s0 * a.tokens * a.out_row, b.rows -= s0 * a.tokens;
    DecodeWork w{reinterpret_cast<float*>(ws), reinterpret_cast<float2*>(ws + d.ml), reinterpret_cast<long long*>(ws + d.base), 0, nullptr};
    int* flags = reinterpret_cast<int*>(ws + d.flags);
    cudaError_t r = cudaSuccess;
    if (paged_decode_tc_takes(b)) {
      const int tokens = paged_decode_tc_rows(b) / b.group;
      w.row_blocks = (b.tokens + tokens - 1) / tokens;
      if (launch_paged_decode_tc(b, std::is_same<T, __half>::value, w, flags, s, &r)) {
        // (a table that names one block of keys: every item lies in one CTA)
        if (r == cudaSuccess && b.max_pages * b.page > 128) r = join_decode<T>(b, w, tokens * b.group, s);
        if (r != cudaSuccess) return r;
        if (b.tokens == 1) continue;  // (what one token sees, all of it sees)
        w.redo = flags;
      }
    }
    w.row_blocks = (a.group * a.tokens + item_rows - 1) / item_rows;
    r = with_decode<T>(b, [&](auto f) { return launch_pdl(f, dim3(kDecCtas), dim3(32 * dec_warps(b)), smem, s, b, w); });
    if (r == cudaSuccess && !w.redo) r = join_decode<T>(b, w, item_rows, s);
    if (r != cudaSuccess) return r;
  }
  return cudaSuccess;
}
template <class T>
cudaError_t launch_prompt(const Paged& a, cudaStream_t s) {
  const int toks = kPpRows / a.group;
  const long long tiles = std::min((long long)a.rows, a.rows / toks + (long long)a.seqs);
  const size_t smem = prompt_smem(a.dim, a.vdim);
  auto go = [&](auto f) { return launch_pdl(f, dim3((unsigned)tiles, a.kv_heads), dim3(kPpThreads), smem, s, a); };
  return a.vdim <= 64 ? go(lm_paged_prompt_kernel<T, 64>) : a.vdim <= 128 ? go(lm_paged_prompt_kernel<T, 128>) : go(lm_paged_prompt_kernel<T, 256>);
}
int status_of(cudaError_t r) { return r == cudaSuccess ? MLLMB200_OK : MLLMB200_CUDA_ERROR; }

__global__ void lm_paged_prep_kernel(int n, const int2* __restrict__ row_sp, const int* __restrict__ table, int ld_table, int page,
                                     int2* __restrict__ row_page, int* __restrict__ lengths) {
  pdl_launch_dependents();
  pdl_wait_prior();
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= n) return;
  const int p = row_sp[b].y, place = p / page;
  row_page[b] = make_int2(table[(size_t)b * ld_table + place], p - place * page);
  lengths[b] = p + 1;
}

}  // namespace

size_t paged_decode_bytes(const Paged& a) { return decode_space(a, std::min(a.seqs, kDecSeqs)).bytes; }
cudaError_t launch_paged_decode(const Paged& a, bool f16, void* workspace, cudaStream_t s) {
  const cudaError_t r = configure_decode();
  if (r != cudaSuccess) return r;
  auto* ws = static_cast<uint8_t*>(workspace);
  return f16 ? launch_decode<__half>(a, ws, s) : launch_decode<__nv_bfloat16>(a, ws, s);
}
cudaError_t launch_paged_prompt(const Paged& a, bool f16, void* workspace, cudaStream_t s) {
  cudaError_t r = cudaSuccess;
  if (launch_paged_prompt_tc(a, f16, workspace, s, &r)) return r;
  r = configure_prompt();
  if (r != cudaSuccess) return r;
  return f16 ? launch_prompt<__half>(a, s) : launch_prompt<__nv_bfloat16>(a, s);
}
cudaError_t launch_paged_prep(cudaStream_t s, int n, const int2* row_sp, const int* table, int ld_table, int page, int2* row_page, int* lengths) {
  return launch_pdl(lm_paged_prep_kernel, dim3((n + 127) / 128), dim3(128), 0, s, n, row_sp, table, ld_table, page, row_page, lengths);
}

}  // namespace lm
}  // namespace mllmb200

using namespace mllmb200;
using namespace mllmb200::lm;

extern "C" {

int mllmb200_lm_pages_append(const mllmb200_lm_pages* pages, const void* k, long long k_row, long long k_head, const void* v, long long v_row,
                             long long v_head, void* stream) {
  Paged a;
  const int st = check_pages(pages, &a);
  if (st != MLLMB200_OK) return st;
  if (!a.seqs || !a.rows) return MLLMB200_OK;
  if (a.kv_heads == 1) k_head = a.dim, v_head = a.vdim;
  if (a.rows == 1) k_row = (long long)a.kv_heads * a.dim, v_row = (long long)a.kv_heads * a.vdim;
  if (!k || !v || !aligned(k, k_row, k_head) || !aligned(v, v_row, v_head)) return MLLMB200_INVALID_ARG;
  const int pieces = a.kv_heads * (a.dim + a.vdim) / 8;
  // (one row a thread while that does not fill the GPU: 64 rows take 2.8 us with one, 5.1 with four; 9476 rows of 4 heads of 128 11.4 and 9)
  const int each = (long long)a.rows * pieces >= 128ll * 16 * kSms ? 4 : 1;
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, dim3((a.rows + each - 1) / each, (pieces + 127) / 128), dim3(128), 0, static_cast<cudaStream_t>(stream), a, k, k_row, k_head, v, v_row,
                      v_head, static_cast<uint16_t*>(pages->k), static_cast<uint16_t*>(pages->v));
  };
  return status_of(each == 4 ? go(lm_pages_append_kernel<4>) : go(lm_pages_append_kernel<1>));
}

int mllmb200_lm_attn_decode_workspace(const mllmb200_lm_pages* pages, const mllmb200_lm_look* look, size_t* bytes) {
  Paged a;
  if (!bytes) return MLLMB200_INVALID_ARG;
  const int st = check_decode(pages, look, &a);
  if (st != MLLMB200_OK) return st;
  *bytes = decode_space(a, std::min(a.seqs, kDecSeqs)).bytes;
  return MLLMB200_OK;
}
int mllmb200_lm_attn_decode(const mllmb200_lm_pages* pages, const mllmb200_lm_look* look, void* workspace, void* stream) {
  Paged a;
  const int st = check_decode(pages, look, &a);
  if (st != MLLMB200_OK) return st;
  if (!a.seqs || !a.rows) return MLLMB200_OK;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u)) return MLLMB200_INVALID_ARG;
  return status_of(launch_paged_decode(a, pages->dtype == MLLMB200_LM_F16, workspace, static_cast<cudaStream_t>(stream)));
}

int mllmb200_lm_attn_prompt_workspace(const mllmb200_lm_pages* pages, const mllmb200_lm_look* look, size_t* bytes) {
  Paged a;
  if (!bytes) return MLLMB200_INVALID_ARG;
  const int st = check_look(pages, look, &a);
  if (st != MLLMB200_OK) return st;
  *bytes = paged_prompt_bytes(a);
  return MLLMB200_OK;
}
int mllmb200_lm_attn_prompt(const mllmb200_lm_pages* pages, const mllmb200_lm_look* look, void* workspace, void* stream) {
  Paged a;
  const int st = check_look(pages, look, &a);
  if (st != MLLMB200_OK) return st;
  if (!a.seqs || !a.rows) return MLLMB200_OK;
  if (paged_prompt_bytes(a) && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u))) return MLLMB200_INVALID_ARG;
  return status_of(launch_paged_prompt(a, pages->dtype == MLLMB200_LM_F16, workspace, static_cast<cudaStream_t>(stream)));
}

int mllmb200_lm_operator_status(void* stream) {
  int status = MLLMB200_OK;
  return read_operator_status(static_cast<cudaStream_t>(stream), &status) == cudaSuccess ? status : MLLMB200_CUDA_ERROR;
}

}  // extern "C"
