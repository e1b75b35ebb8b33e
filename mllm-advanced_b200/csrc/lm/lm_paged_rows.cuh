// Attention of rows over pages on the tensor cores of a warp (mma.sync): any head size, any mask.
#pragma once
#include <algorithm>

#include "lm_paged.h"

namespace mllmb200 {
namespace lm {
namespace {

// o += P V for 16 keys at j0 held as B fragments (mv: address of the first), P = hi + lo of the type (its rounding to 16 bits
// would cost as much as the output's; what two halves keep stands at Num).  EDGE: some of the keys are not seen by some of the
// warp's rows, and what their values hold (infinities, NaN) must not reach those rows through a weight of 0: one token
// of the rows after the other, with the keys that it does not see as zeros.
template <class T, int DV, bool EDGE>
__device__ __forceinline__ void weigh_values(const Paged& a, float (&o)[DV / 8][4], const uint32_t (&hi)[4], const uint32_t (&lo)[4],
                                             uint32_t v_addr, int j0, int lane, const int (&pos)[2], int first, int last) {
  if constexpr (!EDGE) {
#pragma unroll
    for (int n = 0; n < DV / 16; ++n)
      if (n * 16 < a.vdim) {
        uint32_t b[4];
        paged_ldsm_t(b, v_addr + n * 32);
        Num<T>::mma(o[2 * n], hi, b[0], b[1]);
        Num<T>::mma(o[2 * n + 1], hi, b[2], b[3]);
        Num<T>::mma(o[2 * n], lo, b[0], b[1]);
        Num<T>::mma(o[2 * n + 1], lo, b[2], b[3]);
      }
    return;
  } else {
  for (int p = first; p <= last; ++p) {
    uint32_t keep[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = j0 + u * 8 + (lane & 3) * 2;
      keep[u] = (seen_by(a, p, j) ? 0xffffu : 0u) | (seen_by(a, p, j + 1) ? 0xffff0000u : 0u);
    }
#pragma unroll
    for (int n = 0; n < DV / 16; ++n)
      if (n * 16 < a.vdim) {
        uint32_t b[4];
        paged_ldsm_t(b, v_addr + n * 32);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          Num<T>::mma(t, hi, b[2 * u] & keep[0], b[2 * u + 1] & keep[1]);
          Num<T>::mma(t, lo, b[2 * u] & keep[0], b[2 * u + 1] & keep[1]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (pos[i >> 1] == p) o[2 * n + u][i] += t[i];
        }
      }
  }
  }
}

// Scores (base 2) of 16 x 8 N products of one warp for keys from j0 on: scale, bias, mask; the rows' running maxima and sums,
// the weights, times 2^kLift as their sums, in place of the scores.  ALL: every row sees every key.
template <class T, int N, bool ALL>
__device__ __forceinline__ void weigh_keys(const Paged& a, float (&s)[N][4], float (&m)[2], float (&l)[2], float (&alpha)[2], int j0, int lane,
                                           const int (&pos)[2], const float* const (&bias)[2]) {
  float mx[2] = {m[0], m[1]};
  const float scale = a.bias ? 1.0f : a.scale2;
  if (a.bias) {  // (apart: calls without biases would pay for its instructions, long prompts 8 %)
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = j0 + n * 8 + (lane & 3) * 2 + (i & 1), r = i >> 1;
        s[n][i] = fmaf(s[n][i], a.scale2, bias[r] ? in_base2(__ldg(bias[r] + max(0, min(pos[r] - j, a.bias_max)))) : 0.0f);
      }
  }
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + n * 8 + (lane & 3) * 2 + (i & 1), r = i >> 1;
      const float x = s[n][i] * scale;
      s[n][i] = ALL || seen_by(a, pos[r], j) ? x : -INFINITY;
      mx[r] = fmaxf(mx[r], s[n][i]);
    }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
    const float base = mx[r] == -INFINITY ? 0.0f : mx[r];  // (nothing seen yet: every weight is 0)
    alpha[r] = paged_exp2(m[r] - base);
    m[r] = mx[r];
    l[r] *= alpha[r];
    mx[r] = base - Num<T>::kLift;
  }
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[n][i] = paged_exp2(s[n][i] - mx[i >> 1]);
      l[i >> 1] += s[n][i];
    }
}

template <class T>
__device__ __forceinline__ void split_weights(const float (&s0)[4], const float (&s1)[4], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float p0 = (i >> 1 ? s1 : s0)[(i & 1) * 2], p1 = (i >> 1 ? s1 : s0)[(i & 1) * 2 + 1];
    hi[i] = Num<T>::pack(p0, p1);
    const float2 h = Num<T>::unpack(hi[i]);
    lo[i] = Num<T>::pack(p0 - h.x, p1 - h.y);
  }
}

constexpr int kPpRows = 64, kPpKeys = 64, kPpThreads = 256;

size_t prompt_smem(int dim, int vdim) {
  return (size_t)2 * kPpRows * 4 + (size_t)kPpRows * (dim + 8) * 2 + std::max((size_t)2 * kPpKeys * (dim + vdim + 16) * 2, (size_t)kPpRows * vdim * 4);
}

// Which sequence and which of its tiles of `toks` rows a CTA has: {sequence, tile}, sequence -1 past the last one.  All
// threads call it; a sequence's last tiles (the longest) come first.
__device__ __forceinline__ int2 paged_tile(const Paged& a, int index, int toks) {
  __shared__ int2 s_tile;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int2 found = make_int2(-1, 0);
    for (int s0 = 0; s0 < a.seqs; s0 += 32) {
      const int n = s0 + lane < a.seqs ? (paged_rows(a, s0 + lane).y + toks - 1) / toks : 0;
      int up = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, index < up);
      if (hit) {
        const int who = __ffs(hit) - 1;
        found = make_int2(s0 + who, __shfl_sync(0xffffffffu, up, who) - 1 - index);
        break;
      }
      index -= __shfl_sync(0xffffffffu, up, 31);
    }
    if (lane == 0) s_tile = found;
  }
  __syncthreads();
  return s_tile;
}

// The 64 rows (token, query head of kv head kvh) of `ntok` tokens of a sequence from row row0 at position pos0 on, by 256
// threads.  Eight warps: warp w and w + 4 own the same 16 rows and one half each of every block of 64 keys; their states meet
// at the end.  smem: prompt_smem bytes; cta: the barrier of the 256 threads.
template <class T, int DV, class CTA>
__device__ __forceinline__ void paged_prompt_rows(const Paged& a, uint8_t* smem, const CTA& cta, int tid, int seq, int row0, int ntok, int pos0, int kvh) {
  constexpr int kHalf = kPpKeys / 2, kEach = kPpKeys / (kPpThreads / 8);
  const int D = a.dim, p_last = pos0 + ntok - 1;
  const Seen seen = paged_seen<kPpKeys>(a, pos0, p_last);
  const int ldk = D + 8, ldv = a.vdim + 8, warp = tid >> 5, lane = tid & 31, half = warp >> 2, wrow = (warp & 3) * 16;
  float* s_m = reinterpret_cast<float*>(smem);
  float* s_l = s_m + kPpRows;
  T* sQ = reinterpret_cast<T*>(s_l + kPpRows);
  T* sK = sQ + kPpRows * ldk;
  T* sV = sK + 2 * kPpKeys * ldk;
  float* sO = reinterpret_cast<float*>(sK);
  const T* kb = static_cast<const T*>(a.k) + kvh * a.k_head;
  const T* vb = static_cast<const T*>(a.v) + kvh * a.v_head;
  const int cr = tid >> 3, cc = tid & 7;  // copies: eight threads per row of 16-byte pieces
  for (int r = cr; r < kPpRows; r += kPpThreads / 8) {
    const int tok = r / a.group, hg = r - tok * a.group;
    const bool ok = tok < ntok;
    const T* src = static_cast<const T*>(a.q) + (row0 + (ok ? tok : 0)) * a.q_row + (kvh * a.group + hg) * a.q_head;
    for (int c = cc * 8; c < D; c += 64) paged_copy16(smem_u32(sQ + r * ldk + c), ok ? src + c : static_cast<const T*>(a.q), ok);
  }
  auto page_of = [&](int b, int u) {  // page of this thread's row u of block b
    const int j = b < seen.blocks ? block_key<kPpKeys>(seen, b) + cr + u * (kPpThreads / 8) : -1;
    return j >= 0 && seen_by_some(seen, j) ? paged_page(a, seq, j / a.page) : -1;
  };
  int next[kEach];
#pragma unroll
  for (int u = 0; u < kEach; ++u) next[u] = page_of(0, u);
  auto fetch = [&](int b, int buf) {
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int r = cr + u * (kPpThreads / 8), at = (block_key<kPpKeys>(seen, b) + r) % a.page;
      const bool ok = next[u] >= 0;
      const T* ks = ok ? kb + next[u] * a.k_page + at * a.k_row : kb;
      const T* vs = ok ? vb + next[u] * a.v_page + at * a.v_row : vb;
      const uint32_t dk = smem_u32(sK + (buf * kPpKeys + r) * ldk), dv = smem_u32(sV + (buf * kPpKeys + r) * ldv);
      for (int c = cc * 8; c < D; c += 64) paged_copy16(dk + c * 2, ok ? ks + c : kb, ok);
      for (int c = cc * 8; c < a.vdim; c += 64) paged_copy16(dv + c * 2, ok ? vs + c : vb, ok);
      next[u] = page_of(b + 1, u);
    }
    paged_commit();
  };
  if (seen.blocks) fetch(0, 0);
  int pos[2], tok_r[2], hg_r[2];
  const float* bias[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = wrow + (lane >> 2) + i * 8;
    tok_r[i] = r / a.group;
    hg_r[i] = r - tok_r[i] * a.group;
    pos[i] = tok_r[i] < ntok ? pos0 + tok_r[i] : -1;
    bias[i] = a.bias && tok_r[i] < ntok ? a.bias + (size_t)(kvh * a.group + hg_r[i]) * (a.bias_max + 1) : nullptr;
  }
  // positions of this warp's rows
  const int w_first = pos0 + wrow / a.group, w_last = min(p_last, pos0 + (wrow + 15) / a.group);
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[DV / 8][4];
#pragma unroll
  for (int n = 0; n < DV / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
  const int mat = lane >> 3, ml = lane & 7;
  const uint32_t q_addr = smem_u32(sQ + (wrow + (mat & 1) * 8 + ml) * ldk + (mat >> 1) * 8);
  const uint32_t k_addr = smem_u32(sK + (half * kHalf + (mat >> 1) * 8 + ml) * ldk + (mat & 1) * 8);
  const uint32_t v_addr = smem_u32(sV + (half * kHalf + (mat & 1) * 8 + ml) * ldv + (mat >> 1) * 8);

  for (int blk = 0; blk < seen.blocks; ++blk) {
    const int buf = blk & 1, j0 = block_key<kPpKeys>(seen, blk);
    paged_wait<0>();
    cta.sync();
    if (blk + 1 < seen.blocks) fetch(blk + 1, buf ^ 1);
    // values that only some rows see, and that a weight of 0 would not keep from the others
    bool edge = false;
    if (!seen_by_all(a, max(pos0, 0), p_last, j0, j0 + kPpKeys - 1)) {
      for (int r = cr; r < kPpKeys; r += kPpThreads / 8)
        for (int c = cc * 8; c < a.vdim; c += 64) {
          const uint4 x = *reinterpret_cast<const uint4*>(sV + (buf * kPpKeys + r) * ldv + c);
          edge = edge || not_finite2<T>(x.x) || not_finite2<T>(x.y) || not_finite2<T>(x.z) || not_finite2<T>(x.w);
        }
      edge = cta.any(edge);
    }
    if (w_first > p_last) continue;  // (no row of this warp is there)
    const int jw = j0 + half * kHalf;
    float s[kHalf / 8][4];
#pragma unroll
    for (int n = 0; n < kHalf / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll 4
    for (int kk = 0; kk < D; kk += 16) {
      uint32_t qa[4];
      paged_ldsm(qa, q_addr + kk * 2);
#pragma unroll
      for (int n = 0; n < kHalf / 16; ++n) {
        uint32_t b[4];
        paged_ldsm(b, k_addr + ((buf * kPpKeys + n * 16) * ldk + kk) * 2);
        Num<T>::mma(s[2 * n], qa, b[0], b[1]);
        Num<T>::mma(s[2 * n + 1], qa, b[2], b[3]);
      }
    }
    float alpha[2];
    if (w_first >= 0 && seen_by_all(a, w_first, w_last, jw, jw + kHalf - 1)) weigh_keys<T, kHalf / 8, true>(a, s, m, l, alpha, jw, lane, pos, bias);
    else weigh_keys<T, kHalf / 8, false>(a, s, m, l, alpha, jw, lane, pos, bias);
#pragma unroll
    for (int n = 0; n < DV / 8; ++n) o[n][0] *= alpha[0], o[n][1] *= alpha[0], o[n][2] *= alpha[1], o[n][3] *= alpha[1];
#pragma unroll
    for (int kk = 0; kk < kHalf / 16; ++kk) {
      uint32_t hi[4], lo[4];
      split_weights<T>(s[2 * kk], s[2 * kk + 1], hi, lo);
      const uint32_t at = v_addr + (uint32_t)(buf * kPpKeys + kk * 16) * ldv * 2;
      if (!edge) weigh_values<T, DV, false>(a, o, hi, lo, at, jw + kk * 16, lane, pos, 0, 0);
      else weigh_values<T, DV, true>(a, o, hi, lo, at, jw + kk * 16, lane, pos, max(0, w_first), w_last);
    }
  }
  paged_wait<0>();
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    m[r] -= Num<T>::kLift;  // what sums and outputs are relative to
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }
  cta.sync();
  if (half == 1) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = wrow + (lane >> 2) + r * 8;
      if ((lane & 3) == 0) s_m[row] = m[r], s_l[row] = l[r];
      float* so = sO + (size_t)row * a.vdim + (lane & 3) * 2;
#pragma unroll
      for (int n = 0; n < DV / 8; ++n)
        if (n * 8 < a.vdim) *reinterpret_cast<float2*>(so + n * 8) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
    }
  }
  cta.sync();
  if (half == 1) return;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (tok_r[r] >= ntok) continue;
    const int row = wrow + (lane >> 2) + r * 8, h = kvh * a.group + hg_r[r];
    const float sink = a.sink ? in_base2(a.sink[h]) : -INFINITY, mt = fmaxf(fmaxf(m[r], s_m[row]), sink);
    const float base = mt == -INFINITY ? 0.0f : mt, f0 = exp2f(m[r] - base), f1 = exp2f(s_m[row] - base);
    const float sum = l[r] * f0 + s_l[row] * f1 + exp2f(sink - base), inv = pos[r] < 0 ? 0.0f : 1.0f / sum;
    const float* so = sO + (size_t)row * a.vdim + (lane & 3) * 2;
    T* out = static_cast<T*>(a.out) + (row0 + tok_r[r]) * a.out_row + h * a.out_head + (lane & 3) * 2;
#pragma unroll
    for (int n = 0; n < DV / 8; ++n)
      if (n * 8 < a.vdim) {
        const float2 x = *reinterpret_cast<const float2*>(so + n * 8);
        const float v0 = fmaf(o[n][2 * r], f0, x.x * f1) * inv, v1 = fmaf(o[n][2 * r + 1], f0, x.y * f1) * inv;
        *reinterpret_cast<uint32_t*>(out + n * 8) = pos[r] < 0 ? 0u : Num<T>::pack(v0, v1);
      }
  }
}

}  // namespace
}  // namespace lm
}  // namespace mllmb200
