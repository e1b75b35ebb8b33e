// Prompt attention over pages on the 5th-generation tensor cores, heads of 64 or 128 (include/mllmb200_lm.h has the mathematics).
//
// A CTA owns two tiles of 128 rows; a row is (token, query head) of one kv head, so that all heads of a group share every key
// and value that is fetched.  Per block of 128 keys and tile: S = Q K^T into tensor memory, softmax weights P in 16 bits over
// S's own columns, O += P V (64 keys at a time).  While the weights of one tile are made, the products of the other run:
//   warps 0-3, 4-7  weights of tile 0 and 1, a row per thread; O is rescaled (tensor memory) only when a row's maximum has grown by
//                   more than 2^8 (fp16: 2^3) - weights beyond 1 are as exact in 16 bits, and their fp32 sum is kept under the same base
//   warp 8          copies: TMA, pieces of a block that lie in one page, into a ring of keys and one of values
//   warp 9          MMA issue, tensor-memory owner
//   warps 10-11     values of blocks that some rows do not see in full: rows that no row sees (page tails, other sequences' data) are
//                   made zeros; where what only some rows see is not finite, a weight of 0 would not hide it: the tile is
//                   done again row-block by row-block on mma.sync (paged_prompt_rows), which can.
// EXACT: a weight is two numbers of 16 bits, the second what the first one's rounding left, and both meet the values.  Without it the weights'
// rounding (2^-9 of each in bf16, independent) is of the size of the output's own: 2.0e-3 of the 2-norm off instead of 1.5e-3.  The caller
// chooses: half the products more and their making cost 8192 tokens of 16 / 4 heads of 128 a third (284 and 376 us a call), and the engine, whose
// attention over slots carries two numbers, takes EXACT.  Everything else is fp32.
// Measured on a B200: 8192 tokens, 16 / 4 heads of 128, causal: 277-284 us a call with inputs from memory (0.97 PFLOP/s, tensor pipe 52 %
// active; EXACT 60 %), 243 (1.13 PFLOP/s; EXACT 323) back to back in a graph; 2571 rows of five sequences with a window of 512, 12 / 2 heads: 27.  Bound by the chain of a tile: scores, their maximum, weights, product; with two tiles a
// block takes 3900 cycles of which the products need 2048.  Two tiles and not one, since one tile's products hide the other's
// weights; not three, since S and O of two fill tensor memory's 512 columns.  Scores handed over by halves of 64 keys were slower (276 us
// in that graph: twice the waits for the same chain).
#include <algorithm>
#include <atomic>
#include <mutex>

#include "../tcgen05_common.cuh"
#include "lm_paged_rows.cuh"

namespace mllmb200 {
namespace lm {
namespace {

constexpr int kTcKeys = 128, kTcThreads = 384;

template <int D, bool BIAS>
struct TcLayout {
  static constexpr int kTile = 128 * D * 2;  // a block of keys or values, and a tile of queries
  static constexpr int kK = D == 128 ? (BIAS ? 2 : 3) : BIAS ? 3 : 4, kV = D == 128 ? 2 : BIAS ? 3 : 4;  // blocks of keys, of values
  static constexpr int kTable = BIAS ? 30 * 1024 : 0;                                                    // the group's bias tables, if they fit
  static constexpr int kBytes = (2 + kK + kV) * kTile + kTable + 1024;                                   // (queries and ring on 1024 bytes)
};
// Floats from one head's bias table to the next in shared memory: the rows of a warp (all heads of some tokens) read from banks of their own.
__host__ __device__ inline int bias_pitch(int bias_max, int group) {
  const int want = group < 32 ? (32 + group - 1) / group : 1;
  return (bias_max + 32 - want) / 32 * 32 + want;  // at least bias_max + 1
}

template <class T>
__device__ __forceinline__ uint32_t tc_idesc(int n, bool b_mn) {  // fp32 sums, M = 128
  const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
// Operand in the 128-byte swizzle, rows of 64 numbers, groups of 8 rows 1024 bytes apart; `lead`: bytes between chunks of 64
// numbers where those run along M or N (values)
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lead >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map),
               "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
               "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
      "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
      "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

__device__ __forceinline__ uint32_t first_bits(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }

// One row's scores of a block in tensor memory: bias (staged: in shared memory) and mask (written back) and the largest.  first, last: positions of the rows that
// are worked on together.  Loops over columns are short on purpose: a launch starts with a cold instruction cache.
template <bool BIAS>
__device__ __forceinline__ float weigh_block(const Paged& a, uint32_t s_col, const float* bias, bool staged, int pos, int first, int last, int j0) {
  const bool masked = first < 0 || !seen_by_all(a, first, last, j0, j0 + kTcKeys - 1);
  const int hi = pos - j0, lo = a.window ? hi - a.window : -1, kp = a.window ? a.keep - j0 : 0;  // column i: i <= hi and (i > lo or i < kp)
  const bool near = BIAS && first - (j0 + kTcKeys - 1) < a.bias_max;                               // some distance has a bias of its own
  const float far = !BIAS ? 0.0f : staged ? bias[a.bias_max] : in_base2(bias[a.bias_max]);
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 128; c += 64) {
    uint32_t v[2][32];
    tmem_ld32(s_col + c, v[0]);
    tmem_ld32(s_col + c + 32, v[1]);
    tmem_ld_wait();
    if (BIAS) {
      if (near) {
        auto add = [&](auto base2) {
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            uint32_t& x = v[i >> 5][i & 31];
            x = __float_as_uint(fmaf(__uint_as_float(x), a.scale2, base2(bias[max(0, min(hi - c - i, a.bias_max))])));
          }
        };
        if (staged) add([](float b) { return b; });  // (a table in shared memory is in base 2)
        else add(in_base2);
      } else {
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          uint32_t& x = v[i >> 5][i & 31];
          x = __float_as_uint(fmaf(__uint_as_float(x), a.scale2, far));
        }
      }
    }
    if (masked) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = c + h * 32;
        const uint32_t seen = first_bits(hi + 1 - at) & (~first_bits(lo + 1 - at) | first_bits(kp - at));
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (!((seen >> i) & 1u)) v[h][i] = 0xff800000u;
      }
    }
    if (BIAS || masked) {
      tmem_st32(s_col + c, v[0]);
      tmem_st32(s_col + c + 32, v[1]);
    }
    float mx[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) mx[i] = fmaxf(__uint_as_float(v[0][i]), __uint_as_float(v[1][i]));
#pragma unroll
    for (int i = 4; i < 32; ++i) mx[i & 3] = fmaxf(fmaxf(mx[i & 3], __uint_as_float(v[0][i])), __uint_as_float(v[1][i]));
    top = fmaxf(top, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
  }
  if (BIAS || masked) tmem_st_wait();
  return top;
}
// O of the row times alpha, in tensor memory
template <int D>
__device__ __forceinline__ void rescale(uint32_t o_col, float alpha) {
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t o[32];
    tmem_ld32(o_col + c * 32, o);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
    tmem_st32(o_col + c * 32, o);
  }
}
// Two fp32 numbers in a register pair: one instruction for both.
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 pair_parts(uint64_t p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t pair_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x of two numbers up to 127 without the special-function unit, 2^-18 of the result off at most: x = n + f with n whole (the addition
// leaves n + 127 in the low bits of its sum) and |f| <= 1/2; a polynomial of degree 4 for 2^f (least largest relative error, fitted by
// reweighted least squares) times the number whose exponent is n.  Below 2^-126, 0; NaN stays NaN.
__device__ __forceinline__ float2 pair_exp2(uint64_t x) {
  float2 v = pair_parts(x);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.x) : "f"(-127.0f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.y) : "f"(-127.0f));
  x = pair_of(v.x, v.y);
  const uint64_t t = pair_add(x, pair_of(12583039.0f, 12583039.0f));  // 1.5 2^23 + 127
  const uint64_t f = pair_add(x, pair_mul(pair_add(t, pair_of(-12583039.0f, -12583039.0f)), pair_of(-1.0f, -1.0f)));
  uint64_t p = pair_fma(f, pair_of(0.009570102207362652f, 0.009570102207362652f), pair_of(0.05591785907745361f, 0.05591785907745361f));
  p = pair_fma(p, f, pair_of(0.240247443318367f, 0.240247443318367f));
  p = pair_fma(p, f, pair_of(0.6931217908859253f, 0.6931217908859253f));
  p = pair_fma(p, f, pair_of(0.9999992847442627f, 0.9999992847442627f));
  const float2 n = pair_parts(t);
  return pair_parts(pair_mul(p, pair_of(__uint_as_float(__float_as_uint(n.x) << 23), __uint_as_float(__float_as_uint(n.y) << 23))));
}

// weights 2^(score scale + base) over the scores' columns: for the 64 keys whose scores lay there 32 columns of weights in 16 bits and, EXACT, 32
// of what their rounding left, in 16 bits too; their sum.  ready(h): those of keys 64 h and on are there.  The special-function unit takes 1024 cycles for a tile's exponentials, as long as a
// product of a tile; every kPoly-th pair goes through the other pipes instead.
constexpr int kPoly = 4;
template <class T, bool EXACT, class F>
__device__ __forceinline__ float put_weights(uint32_t s_col, float scale, float base, F ready) {
  const uint64_t scale2 = pair_of(scale, scale), base2 = pair_of(base, base);
  uint64_t sum[2] = {0, 0};
#pragma unroll 1
  for (int c = 0; c < 128; c += 64) {
    uint32_t v[2][32];
    tmem_ld32(s_col + c, v[0]);
    tmem_ld32(s_col + c + 32, v[1]);
    tmem_ld_wait();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t hi[16], lo[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint64_t x = pair_fma(pair_of(__uint_as_float(v[h][2 * i]), __uint_as_float(v[h][2 * i + 1])), scale2, base2);
        float2 e;
        if (i % kPoly == kPoly - 1) {
          e = pair_exp2(x);
        } else {
          const float2 y = pair_parts(x);
          e = make_float2(paged_exp2(y.x), paged_exp2(y.y));
        }
        sum[i & 1] = pair_add(sum[i & 1], pair_of(e.x, e.y));
        hi[i] = Num<T>::pack(e.x, e.y);
        if constexpr (EXACT) {
          const float2 up = Num<T>::unpack(hi[i]);
          lo[i] = Num<T>::pack(e.x - up.x, e.y - up.y);
        }
      }
      tmem_st16(s_col + c + h * 16, hi);
      if constexpr (EXACT) tmem_st16(s_col + c + 32 + h * 16, lo);
    }
    tmem_st_wait();
    ready(c / 64);
  }
  const float2 total = pair_parts(pair_add(sum[0], sum[1]));
  return total.x + total.y;
}

// Few rows and long contexts: `parts` CTAs (gridDim.y) share a pair of tiles' blocks and leave {maximum, sum} and unnormalized outputs
// [CTA][part][256 rows]; flags [CTA][part]: 1 where the part has been done again in full (see below).
struct PromptSplit {
  float* part_o;
  float2* part_ml;
  int *flags, parts;
};

struct TcBarriers {
  uint64_t q_full, k_full[4], k_free[4], v_full[4], v_free[4], v_fixed[4], s_full[2], p_ready[2][2], o_done[2];
};

template <class T, int D, bool BIAS, bool EXACT>
__global__ void __launch_bounds__(kTcThreads, 1) lm_paged_prompt_tc_kernel(const __grid_constant__ Paged a, const __grid_constant__ CUtensorMap qmap,
                                                                           const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                                                           int piece, PromptSplit w) {
  using L = TcLayout<D, BIAS>;
  extern __shared__ uint8_t tc_smem_raw[];
  __shared__ TcBarriers bars;
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_bad, s_gave_up;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t smem0 = (smem_u32(tc_smem_raw) + 1023u) & ~1023u, keys0 = smem0 + 2 * L::kTile, values0 = keys0 + L::kK * L::kTile;
  if (tid < 3) tma_prefetch_map(tid == 0 ? &qmap : tid == 1 ? &kmap : &vmap);
  pdl_wait_prior();
  const int toks = 128 / a.group, kvh = blockIdx.x % a.kv_heads;
  const int2 tile = paged_tile(a, blockIdx.x / a.kv_heads, 2 * toks);
  if (tile.x < 0) return;
  const int2 seq_rows = paged_rows(a, tile.x);
  const int row0 = seq_rows.x + tile.y * 2 * toks, ntok = min(2 * toks, seq_rows.y - tile.y * 2 * toks);
  const int pos0 = paged_length(a, tile.x) - seq_rows.y + tile.y * 2 * toks, p_last = pos0 + ntok - 1;
  const Seen seen = paged_seen<kTcKeys>(a, pos0, p_last);
  const int b0 = (int)((long long)seen.blocks * blockIdx.y / w.parts), nt = (int)((long long)seen.blocks * (blockIdx.y + 1) / w.parts) - b0;  // this CTA's blocks
  const int tiles = ntok > toks ? 2 : 1;
  if (tid == 0) {
    mbar_init(&bars.q_full, 1);
    for (int i = 0; i < L::kK; ++i) mbar_init(&bars.k_full[i], 1), mbar_init(&bars.k_free[i], 1);
    for (int i = 0; i < L::kV; ++i) mbar_init(&bars.v_full[i], 1), mbar_init(&bars.v_free[i], 1), mbar_init(&bars.v_fixed[i], 2);
    for (int i = 0; i < 2; ++i) mbar_init(&bars.s_full[i], 1), mbar_init(&bars.p_ready[i][0], 4), mbar_init(&bars.p_ready[i][1], 4), mbar_init(&bars.o_done[i], 1);
    s_bad = s_gave_up = 0;
    mbar_fence_init();
  }
  if (warp == 9) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  const int pitch = BIAS ? bias_pitch(a.bias_max, a.group) : 0;
  const bool staged = BIAS && (size_t)pitch * a.group * 4 <= (size_t)L::kTable;
  float* table = reinterpret_cast<float*>(tc_smem_raw + (values0 + L::kV * L::kTile - smem_u32(tc_smem_raw)));
  if (staged)
    for (int h = warp; h < a.group; h += kTcThreads / 32)
      for (int i = lane; i <= a.bias_max; i += 32) table[h * pitch + i] = in_base2(a.bias[(size_t)(kvh * a.group + h) * (a.bias_max + 1) + i]);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // (not before this CTA has its tensor memory, and not taken before the kernels in front have ended: a kernel that takes some of it and
  // then waits for another must not keep that one from taking its own)
  pdl_launch_dependents();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
  auto turn = [](int j, int n) { return (uint32_t)(j / n) & 1u; };  // parity of a ring's pass
  auto partly = [&](int j) {  // some row does not see some key of block j
    const int j0 = block_key<kTcKeys>(seen, b0 + j);
    return pos0 < 0 || !seen_by_all(a, pos0, p_last, j0, j0 + kTcKeys - 1);
  };
  auto bounded = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_bounded(bar, parity, 1ll << 31, a.timeout); };
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    if (s_gave_up) return false;
    if (bounded(bar, parity)) return true;
    s_gave_up = 1;
    return false;
  };

  if (warp >= 8) {
    if (warp == 8) {
      // ---------------------------------------------------------- copies
      if (nt) {
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars.q_full, (uint32_t)(tiles * toks * a.group * D * 2));
          for (int t = 0; t < tiles; ++t)
            for (int c = 0; c < D / 64; ++c) tma_load_3d(smem0 + t * L::kTile + c * 16384, &qmap, c * 64, kvh * a.group, row0 + t * toks, &bars.q_full);
        }
        const int pieces = kTcKeys / piece;
        int n_k = 0, n_v = 0;
        bool ok = true;
        auto page_of = [&](int j) {  // lane i: page of piece i of block j, a.pages (zeros) where nothing of it is seen
          int page = a.pages;
          if (j < nt && lane < pieces) {
            const int key = block_key<kTcKeys>(seen, b0 + j) + lane * piece;
            if (key <= seen.last && (key + piece > seen.lo || key < seen.head)) {
              const int p = paged_page(a, tile.x, key / a.page);
              if (p >= 0) page = p;
            }
          }
          return page;
        };
        int pages = page_of(0);
        for (int j = 0; j < nt && ok; ++j) {
          const int next = page_of(j + 1), j0 = block_key<kTcKeys>(seen, b0 + j);
          auto copy = [&](const CUtensorMap* map, uint32_t block, uint64_t* full) {
            if (lane == 0) mbar_arrive_expect_tx(full, L::kTile);
            __syncwarp();
            if (lane < pieces) {
              const int at = (j0 + lane * piece) % a.page;
#pragma unroll
              for (int c = 0; c < D / 64; ++c) tma_load_4d(block + lane * piece * 128 + c * 16384, map, c * 64, at, kvh, pages, full);
            }
            __syncwarp();
          };
          const int ks = j % L::kK, vs = j % L::kV;
          if (j >= L::kK) ok = __all_sync(0xffffffffu, wait(&bars.k_free[ks], turn(j, L::kK) ^ 1u));
          if (!ok) break;
          copy(&kmap, keys0 + ks * L::kTile, &bars.k_full[ks]);
          ++n_k;
          if (j >= L::kV) ok = __all_sync(0xffffffffu, wait(&bars.v_free[vs], turn(j, L::kV) ^ 1u));
          if (!ok) break;
          copy(&vmap, values0 + vs * L::kTile, &bars.v_full[vs]);
          ++n_v;
          pages = next;
        }
        if (!ok) {  // nothing in flight when the CTA leaves
          bounded(&bars.q_full, 0);
          for (int j = max(0, n_k - L::kK); j < n_k; ++j) bounded(&bars.k_full[j % L::kK], turn(j, L::kK));
          for (int j = max(0, n_v - L::kV); j < n_v; ++j) bounded(&bars.v_full[j % L::kV], turn(j, L::kV));
        }
      }
    } else if (warp == 9) {
      // ---------------------------------------------------------- MMA issue
      if (nt) {
        const bool issuer = elect_one_sync();
        const uint32_t idesc_s = tc_idesc<T>(kTcKeys, false), idesc_o = tc_idesc<T>(D, true);
        auto all_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
        auto scores = [&](int t, int j, bool last) {
          if (issuer) {
            const uint64_t q = tc_desc(smem0 + t * L::kTile, 16), k = tc_desc(keys0 + j % L::kK * L::kTile, 16);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const uint64_t off = (uint64_t)((ks / 4) * 1024 + (ks % 4) * 2);
              tc_mma_f16(tmem + t * 128, q + off, k + off, idesc_s, ks > 0);
            }
            tc_commit(&bars.s_full[t]);
            if (last) tc_commit(&bars.k_free[j % L::kK]);
          }
          __syncwarp();
        };
        bool ok = all_wait(&bars.q_full, 0) && all_wait(&bars.k_full[0], 0);
        if (ok) {
          tc_fence_after();
          for (int t = 0; t < tiles; ++t) scores(t, 0, t == tiles - 1);
        }
        for (int j = 0; j < nt && ok; ++j) {
          // (what is there long before the weights is waited for before them)
          ok = all_wait(&bars.v_full[j % L::kV], turn(j, L::kV)) && all_wait(&bars.v_fixed[j % L::kV], turn(j, L::kV));
          if (ok && j + 1 < nt) ok = all_wait(&bars.k_full[(j + 1) % L::kK], turn(j + 1, L::kK));
          for (int t = 0; t < tiles && ok; ++t) {
            for (int h = 0; h < 2 && ok; ++h) {  // keys 64 h and on: the products of the first 64 run while the other weights are made
              ok = all_wait(&bars.p_ready[t][h], (uint32_t)j & 1u);
              if (!ok) break;
              tc_fence_after();
              if (issuer) {
                const uint64_t v = tc_desc(values0 + j % L::kV * L::kTile, 16384);
#pragma unroll
                for (int ks = 0; ks < (EXACT ? 8 : 4); ++ks)  // the weights, then what their rounding left
                  tc_mma_f16_ts(tmem + 256 + t * D, tmem + t * 128 + h * 64 + ks * 8, v + (uint64_t)((h * 4 + (ks & 3)) * 128), idesc_o, j > 0 || h > 0 || ks > 0);
                if (h == 1 && t == tiles - 1) tc_commit(&bars.v_free[j % L::kV]);
                if (h == 1 && j == nt - 1) tc_commit(&bars.o_done[t]);
              }
              __syncwarp();
            }
            if (!ok) break;
            if (j + 1 < nt) scores(t, j + 1, t == tiles - 1);
          }
        }
      }
    } else {
      // ---------------------------------------------------------- values that not every row sees
      bool ok = true;
      for (int j = 0; j < nt && ok; ++j) {
        ok = wait(&bars.v_full[j % L::kV], turn(j, L::kV));
        if (!ok) break;
        const int j0 = block_key<kTcKeys>(seen, b0 + j);
        const uint32_t block = values0 + j % L::kV * L::kTile;
        bool bad = false;
        for (int r = partly(j) ? tid - 320 : kTcKeys; r < kTcKeys; r += 64) {
          const bool some = seen_by_some(seen, j0 + r);
          if (some && pos0 >= 0 && seen_by_all(a, pos0, p_last, j0 + r, j0 + r)) continue;
          for (int c = 0; c < D / 8; ++c) {
            const uint32_t at = block + (c / 8) * 16384 + r * 128 + (((c % 8) ^ (r & 7)) * 16);
            if (some) {
              uint4 x;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
              bad = bad || not_finite2<T>(x.x) || not_finite2<T>(x.y) || not_finite2<T>(x.z) || not_finite2<T>(x.w);
            } else {
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0u) : "memory");
            }
          }
        }
        if (bad) s_bad = 1;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.v_fixed[j % L::kV]);
      }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
      tc_fence_after();
      tmem_dealloc(tmem, 512);
    }
    return;
  }

  // ------------------------------------------------------------ weights: one row per thread
  {
    const int t = warp >> 2, r = tid & 127, tok = r / a.group, hg = r - tok * a.group, head = kvh * a.group + hg;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_col = tmem + t * 128 + lanes, o_col = tmem + 256 + t * D + lanes;
    const bool live = tok < toks && t * toks + tok < ntok;
    const int pos = live ? pos0 + t * toks + tok : -1;
    const int first = pos0 + t * toks, last = min(p_last, first + toks - 1);  // of this tile
    // (a row that is not there reads the first one's)
    const float* bias = !BIAS ? nullptr : staged ? table + (live ? hg * pitch : 0) : a.bias + (size_t)(live ? head : 0) * (a.bias_max + 1);
    const float sink = a.sink && live ? in_base2(a.sink[head]) : -INFINITY;
    const float scale = BIAS ? 1.0f : a.scale2, grown = Num<T>::kLag / scale;  // BIAS: scores are scaled before their maximum
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    const int n = t < tiles ? nt : 0;
    for (int j = 0; j < n; ++j) {
      ok = ok && __all_sync(0xffffffffu, wait(&bars.s_full[t], (uint32_t)j & 1u));
      tc_fence_after();
      const float top = weigh_block<BIAS>(a, s_col, bias, staged, pos, first, last, block_key<kTcKeys>(seen, b0 + j));
      if (__any_sync(0xffffffffu, live && top > m + grown)) {
        const float m_new = fmaxf(m, top), alpha = m_new == -INFINITY ? 1.0f : paged_exp2((m - m_new) * scale);
        m = m_new;
        if (j > 0) {  // (the products before S of this block are done)
          l *= alpha;
          rescale<D>(o_col, alpha);
        }
      }
      l += put_weights<T, EXACT>(s_col, scale, m == -INFINITY ? 0.0f : fmaf(-m, scale, Num<T>::kLift), [&](int h) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_ready[t][h]);
      });
    }
    if (n) ok = ok && __all_sync(0xffffffffu, wait(&bars.o_done[t], 0));
    tc_fence_after();
    const bool split = w.parts > 1;
    const size_t at = ((size_t)blockIdx.x * w.parts + blockIdx.y) * 256 + tid;  // tid: tile and row
    T* out = static_cast<T*>(a.out) + (row0 + t * toks + tok) * a.out_row + head * a.out_head;
    if (n == 0 && live) {
      if (split) {
        w.part_ml[at] = make_float2(-INFINITY, 0.0f);
      } else {
        for (int d = 0; d < D; d += 8) *reinterpret_cast<uint4*>(out + d) = make_uint4(0, 0, 0, 0);
      }
    }
    if (n) {
      const float ref = fmaf(m, scale, -Num<T>::kLift);  // what sums and outputs are relative to (base 2)
      const float total = l + (split ? 0.0f : paged_exp2(sink - (m == -INFINITY ? 0.0f : ref))), inv = pos < 0 ? 0.0f : 1.0f / total;
      if (split && live) w.part_ml[at] = make_float2(ref, l);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(o_col + c * 32, o);
        tmem_ld_wait();
        if (!live || !ok) continue;
        if (split) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            reinterpret_cast<uint4*>(w.part_o + at * D + c * 32)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              y[k] = pos < 0 ? 0u : Num<T>::pack(__uint_as_float(o[8 * i + 2 * k]) * inv, __uint_as_float(o[8 * i + 2 * k + 1]) * inv);
            *reinterpret_cast<uint4*>(out + c * 32 + i * 8) = make_uint4(y[0], y[1], y[2], y[3]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && w.parts > 1) w.flags[(size_t)blockIdx.x * w.parts + blockIdx.y] = s_bad;
  if (!s_bad) return;
  struct Cta {
    __device__ void sync() const { asm volatile("bar.sync 1, 256;" ::: "memory"); }
    __device__ bool any(bool v) const {
      int r;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 256, p;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((int)v) : "memory");
      return r != 0;
    }
  };
  const Cta cta{};
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tc_smem_raw) + 1023) & ~(uintptr_t)1023);
  const int few = kPpRows / a.group;
  for (int t = 0; t < ntok; t += few) {
    cta.sync();
    paged_prompt_rows<T, D>(a, smem, cta, tid, tile.x, row0 + t, min(few, ntok - t), pos0 + t, kvh);
  }
}

// grid (CTAs of the kernel above, 8): a warp joins the parts of four rows.
template <class T, int D>
__global__ void __launch_bounds__(256) lm_paged_prompt_join_kernel(Paged a, PromptSplit w) {
  pdl_launch_dependents();
  pdl_wait_prior();
  const int toks = 128 / a.group, kvh = blockIdx.x % a.kv_heads, lane = threadIdx.x & 31;
  const int2 tile = paged_tile(a, blockIdx.x / a.kv_heads, 2 * toks);
  if (tile.x < 0) return;
  for (int i = 0; i < w.parts; ++i)
    if (w.flags[(size_t)blockIdx.x * w.parts + i]) return;  // done there
  const int2 rows = paged_rows(a, tile.x);
  const int first = tile.y * 2 * toks, pos0 = paged_length(a, tile.x) - rows.y + first;
  for (int u = 0; u < 4; ++u) {
    const int i = blockIdx.y * 32 + (threadIdx.x >> 5) * 4 + u, r = i & 127, tok = (i >> 7) * toks + r / a.group, head = kvh * a.group + r % a.group;
    if (r / a.group >= toks || first + tok >= rows.y) continue;
    auto at = [&](int p) { return ((size_t)blockIdx.x * w.parts + p) * 256 + i; };
    const float2 ml = lane < w.parts ? w.part_ml[at(lane)] : make_float2(-INFINITY, 0.0f);
    const float sink = a.sink ? in_base2(a.sink[head]) : -INFINITY;
    float mx = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mx = fmaxf(mx, sink);
    const float base = mx == -INFINITY ? 0.0f : mx, f = ml.y == 0.0f ? 0.0f : exp2f(ml.x - base);
    float sum = f * ml.y, v[D / 32] = {};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    for (int p = 0; p < w.parts; ++p) {
      const float fp = __shfl_sync(0xffffffffu, f, p);
      if (fp == 0.0f) continue;  // (an empty part has left no output)
      const float* part = w.part_o + at(p) * D + lane * (D / 32);
#pragma unroll
      for (int k = 0; k < D / 32; k += 2) {
        const float2 x = *reinterpret_cast<const float2*>(part + k);
        v[k] = fmaf(fp, x.x, v[k]), v[k + 1] = fmaf(fp, x.y, v[k + 1]);
      }
    }
    const float inv = 1.0f / (sum + exp2f(sink - base));
    T* out = static_cast<T*>(a.out) + (rows.x + first + tok) * a.out_row + head * a.out_head + lane * (D / 32);
#pragma unroll
    for (int k = 0; k < D / 32; k += 2) *reinterpret_cast<uint32_t*>(out + k) = pos0 + tok < 0 ? 0u : Num<T>::pack(v[k] * inv, v[k + 1] * inv);
  }
}

// ------------------------------------------------------------------------------------------ a few tokens per sequence
// What bounds this is the stream of keys and values (64 KB a block of 128 keys for heads of 128), as long as a block's work stays
// shorter than its way from memory.  So the keys are the wide side of both products: S^T = K Q^T has a key per lane and an item's rows
// (all heads of a kv head, of up to 64 / group tokens) as its 16, 32 or 64 columns, and O^T += V^T P^T a value's number per lane.
// Every thread of the four warps has its own key; a row's maximum is looked for across threads only when some score has
// outgrown the one in use by more than 2^8 (fp16: 2^3), and sums are added up across threads at an item's end.  Weights enter as two halves of
// 16 bits (Num says what they keep).  A CTA walks an even share of all blocks, copies running ahead over the ends of items:
//   warps 0-3        weights
//   warp 4, 5, 6     copies; MMA issue (scores a block ahead); values that not every row sees
// Five tokens of 32 contexts of 8-12 k, 16 / 4 heads of 128: 107-124 us of 129 in all, 658 MB at 5.3-6.1 TB/s (rows as lanes: 158-197, three
// quarters of the lanes without a row).  One token of 64 contexts of 200-1100: 27, of which 4.7 pass before the first copy lands.
struct Share {  // a CTA's part of an item
  int seq, kvh, row0, ntok, blk0, n, p_first, p_last;
  bool begins, whole;
  Seen all;  // what the sequence's rows see: the blocks; the item's own rows are at p_first .. p_last
};
__device__ __forceinline__ Share share_at(const Paged& a, const int* base, const int* lengths, int row_blocks, int tpi, int b, int end) {
  Share g;
  const int items = a.kv_heads * row_blocks;
  int s = 0;
  for (int step = kDecSeqs / 2; step; step /= 2)
    if (s + step < a.seqs && base[s + step] * items <= b) s += step;
  g.seq = s;
  const int len = lengths[s];
  g.all = paged_seen<kTcKeys>(a, len - a.tokens, len - 1);
  const int in_seq = b - base[s] * items, item = in_seq / g.all.blocks, rb = item % row_blocks;
  g.blk0 = in_seq - item * g.all.blocks;
  g.n = min(end - b, g.all.blocks - g.blk0);
  g.kvh = item / row_blocks;
  const int2 rows = paged_rows(a, s);
  g.row0 = rows.x + rb * tpi;
  g.ntok = min(min(tpi, a.tokens - rb * tpi), max(0, rows.y - rb * tpi));
  g.p_first = len - a.tokens + rb * tpi;
  g.p_last = g.p_first + g.ntok - 1;
  g.begins = g.blk0 == 0;
  g.whole = g.begins && g.n == g.all.blocks;
  return g;
}
// Place in a ring of n: slot and the parity of its pass.
struct Ring {
  int slot = 0, count = 0;
  uint32_t pass = 0;
  __device__ __forceinline__ void next(int n) {
    ++count;
    if (++slot == n) slot = 0, pass ^= 1u;
  }
};
constexpr int kDecThreads = 256;

template <int D, int NP>
struct DecLayout {
  static constexpr int kTile = 128 * D * 2;     // a block of keys or values
  static constexpr int kQ = NP * D * 2;         // an item's queries
  static constexpr int kP = 128 * NP * 2;       // weights of a block, one half
  static constexpr int kBufs = NP == 16 ? 2 : 1;  // places for queries and for weights: with more rows keys and values need the room more
  static constexpr int kFixed = 1024 + kBufs * (kQ + 2 * kP);
  static constexpr int kBlocks = (232448 - 7168 - kFixed) / kTile < 12 ? (232448 - 7168 - kFixed) / kTile : 12;  // (7168: the static part)
  static constexpr int kV = kBlocks / 2, kK = kBlocks - kV;
  static constexpr int kBytes = kFixed + kBlocks * kTile;
  static constexpr int kColumns = NP <= 16 ? 64 : NP <= 32 ? 128 : 256;  // of tensor memory: S twice, O
  static constexpr uint64_t kSwizzle = NP == 16 ? 6 : NP == 32 ? 4 : 2;  // rows of 32, 64, 128 bytes
};
template <int D, int NP>
struct DecBarriers {
  using L = DecLayout<D, NP>;
  uint64_t q_full[2], q_free[2], k_full[L::kK], k_free[L::kK], v_full[L::kV], v_free[L::kV], v_fixed[L::kV], s_full[2], p_ready[2], p_free[2], o_free;
};

template <class T, int D, int NP, bool BIAS>
__global__ void __launch_bounds__(kDecThreads, 1) lm_paged_decode_tc_kernel(const __grid_constant__ Paged a, const __grid_constant__ CUtensorMap qmap,
                                                                            const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                                                            DecodeWork w, int* flags, int piece, int tpi) {
  using L = DecLayout<D, NP>;
  constexpr int kC = NP < 32 ? NP : 32;  // columns handled at a time
  extern __shared__ uint8_t tc_smem_raw[];
  __shared__ DecBarriers<D, NP> bars;
  __shared__ int s_base[kDecSeqs + 1], s_len[kDecSeqs];
  __shared__ float s_max[4][NP];
  __shared__ __align__(16) float s_ref[NP], s_alpha[NP], s_base2[NP], s_far[BIAS ? NP : 1];  // the rows' maxima by warp; the one in use, times scale (base 2); what is added to scores; the bias of far keys
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_bad, s_gave_up;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  // keys, values, weights [kBufs][halves][128 keys][NP], queries [kBufs][D / 64][NP][64]
  const uint32_t keys0 = (smem_u32(tc_smem_raw) + 1023u) & ~1023u, values0 = keys0 + L::kK * L::kTile, p0 = values0 + L::kV * L::kTile, q0 = p0 + L::kBufs * 2 * L::kP;
  constexpr int kB = L::kBufs;
  const int item_rows = tpi * a.group;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i)
      mbar_init(&bars.q_full[i], 1), mbar_init(&bars.q_free[i], 1), mbar_init(&bars.s_full[i], 1), mbar_init(&bars.p_ready[i], 4), mbar_init(&bars.p_free[i], 1);
    for (int i = 0; i < L::kK; ++i) mbar_init(&bars.k_full[i], 1), mbar_init(&bars.k_free[i], 1);
    for (int i = 0; i < L::kV; ++i) mbar_init(&bars.v_full[i], 1), mbar_init(&bars.v_free[i], 1), mbar_init(&bars.v_fixed[i], 1);
    mbar_init(&bars.o_free, 4);
    s_bad = s_gave_up = 0;
    mbar_fence_init();
  }
  if (tid < 3) tma_prefetch_map(tid == 0 ? &qmap : tid == 1 ? &kmap : &vmap);
  pdl_wait_prior();
  if (warp == 5) {
    tmem_alloc(&s_tmem, L::kColumns);
    tmem_relinquish();
  }
  sum_blocks<kTcKeys, kDecThreads>(a, s_base, s_len);
  if (blockIdx.x == 0)
    for (int i = tid; i <= a.seqs; i += kDecThreads) w.base[i] = s_base[i];
  for (int s = blockIdx.x; s < a.seqs; s += gridDim.x) {  // sequences without keys
    if (s_base[s + 1] != s_base[s]) continue;
    const int2 rows = paged_rows(a, s);
    for (int i = tid; i < min(rows.y, a.tokens) * a.heads * (D / 8); i += kDecThreads) {
      const int c = i % (D / 8), h = i / (D / 8) % a.heads, t = i / (D / 8) / a.heads;
      *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (rows.x + t) * a.out_row + h * a.out_head + c * 8) = make_uint4(0, 0, 0, 0);
    }
  }
  const int total = s_base[a.seqs] * a.kv_heads * w.row_blocks, shares = min((int)gridDim.x, total);  // (every one of them has something)
  const bool some = (int)blockIdx.x < shares;
  const int start = some ? (int)((long long)total * blockIdx.x / shares) : 0, end = some ? (int)((long long)total * (blockIdx.x + 1) / shares) : 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();  // (as above)
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
  auto bounded = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_bounded(bar, parity, 1ll << 31, a.timeout); };
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    if (s_gave_up) return false;
    if (bounded(bar, parity)) return true;
    s_gave_up = 1;
    return false;
  };
  auto all_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
  struct Place {  // of a role in the list of blocks
    int b, i, sg;
    Share g;
  } p{start, 0, 0, {}};
  auto enter = [&](Place& q) {  // block q.b: its share
    if (q.i == 0) q.g = share_at(a, s_base, s_len, w.row_blocks, tpi, q.b, end);
  };
  auto leave = [&](Place& q) {
    ++q.b;
    if (++q.i == q.g.n) q.i = 0, ++q.sg;
  };

  if (warp == 4) {
    // ------------------------------------------------------------ copies
    const int pieces = kTcKeys / piece;
    bool ok = true;
    Ring kr, vr;
    while (p.b < end && ok) {
      enter(p);
      if (p.i == 0) {
        const int qb = p.sg % kB;
        if (p.sg >= kB) ok = all_wait(&bars.q_free[qb], (uint32_t)(p.sg / kB - 1) & 1u);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars.q_full[qb], (uint32_t)(item_rows * D * 2));
          for (int c = 0; c < D / 64; ++c) tma_load_3d(q0 + qb * L::kQ + c * NP * 128, &qmap, c * 64, p.g.kvh * a.group, p.g.row0, &bars.q_full[qb]);
        }
        __syncwarp();
      }
      // lane l: row inside its page and page of piece l of the share's block i, a.pages (zeros) where nothing of it is seen
      auto piece_of = [&](int i) {
        const int key = block_key<kTcKeys>(p.g.all, p.g.blk0 + i) + lane * piece, place = key / a.page;
        int page = a.pages;
        if (i < p.g.n && lane < pieces && key <= p.g.all.last && (key + piece > p.g.all.lo || key < p.g.all.head)) {
          const int q = paged_page(a, p.g.seq, place);
          if (q >= 0) page = q;
        }
        return make_int2(key - place * a.page, page);
      };
      const int2 there = piece_of(p.i);
      const int inside = there.x, page = there.y;
      auto copy = [&](const CUtensorMap* map, uint32_t block, uint64_t* full) {
        if (lane == 0) mbar_arrive_expect_tx(full, L::kTile);
        __syncwarp();
        if (lane < pieces) {
#pragma unroll
          for (int c = 0; c < D / 64; ++c) tma_load_4d(block + lane * piece * 128 + c * 16384, map, c * 64, inside, p.g.kvh, page, full);
        }
        __syncwarp();
      };
      if (kr.count >= L::kK) ok = all_wait(&bars.k_free[kr.slot], kr.pass ^ 1u);
      if (!ok) break;
      copy(&kmap, keys0 + kr.slot * L::kTile, &bars.k_full[kr.slot]);
      kr.next(L::kK);
      if (vr.count >= L::kV) ok = all_wait(&bars.v_free[vr.slot], vr.pass ^ 1u);
      if (!ok) break;
      copy(&vmap, values0 + vr.slot * L::kTile, &bars.v_full[vr.slot]);
      vr.next(L::kV);
      leave(p);
    }
    if (!ok) {  // nothing in flight when the CTA leaves
      for (int i = max(0, kr.count - L::kK); i < kr.count; ++i) bounded(&bars.k_full[i % L::kK], (uint32_t)(i / L::kK) & 1u);
      for (int i = max(0, vr.count - L::kV); i < vr.count; ++i) bounded(&bars.v_full[i % L::kV], (uint32_t)(i / L::kV) & 1u);
      for (int i = max(0, p.sg + 1 - kB); i <= p.sg; ++i) bounded(&bars.q_full[i % kB], (uint32_t)(i / kB) & 1u);
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------ MMA issue
    const bool issuer = elect_one_sync();
    const uint32_t idesc_s = tc_idesc<T>(NP, false), idesc_o = tc_idesc<T>(NP, true) | (1u << 15);  // both operands of O^T run along M, N
    bool ok = true;
    Place ps = p;
    Ring kr, vr;
    auto scores = [&]() {  // of block kr.count
      if (ps.b >= end || !ok) return;
      enter(ps);
      if (ps.i == 0) ok = all_wait(&bars.q_full[ps.sg % kB], (uint32_t)(ps.sg / kB) & 1u);
      ok = ok && all_wait(&bars.k_full[kr.slot], kr.pass);
      if (!ok) return;
      tc_fence_after();
      if (issuer) {
        const uint64_t k = tc_desc(keys0 + kr.slot * L::kTile, 16), q = tc_desc(q0 + ps.sg % kB * L::kQ, 16);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          tc_mma_f16(tmem + (kr.count & 1) * NP, k + (uint64_t)((ks / 4) * 1024 + (ks % 4) * 2), q + (uint64_t)((ks / 4) * NP * 8 + (ks % 4) * 2), idesc_s, ks > 0);
        tc_commit(&bars.s_full[kr.count & 1]);
        tc_commit(&bars.k_free[kr.slot]);
        if (ps.i == ps.g.n - 1) tc_commit(&bars.q_free[ps.sg % kB]);
      }
      __syncwarp();
      kr.next(L::kK);
      leave(ps);
    };
    scores();
    scores();
    while (p.b < end && ok) {
      enter(p);
      const int r = vr.count;
      ok = all_wait(&bars.v_full[vr.slot], vr.pass) && all_wait(&bars.v_fixed[vr.slot], vr.pass);
      if (ok && p.i == 0 && p.sg > 0) ok = all_wait(&bars.o_free, (uint32_t)(p.sg - 1) & 1u);  // the last share's output has been read
      ok = ok && all_wait(&bars.p_ready[r & 1], (uint32_t)(r >> 1) & 1u);
      if (!ok) break;
      tc_fence_after();
      if (issuer) {
        constexpr uint32_t kStep = NP * 2 * 16 / 16;  // 16 keys of weights, in 16 bytes
        const uint64_t v = tc_desc(values0 + vr.slot * L::kTile, 16384);
        const uint64_t hi = (uint64_t)(((p0 + r % kB * 2 * L::kP) >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(NP * 16 >> 4) << 32) | (1ull << 46) | (L::kSwizzle << 61);
#pragma unroll
        for (int ks = 0; ks < kTcKeys / 8; ++ks)  // the upper halves, then the lower
          tc_mma_f16(tmem + 2 * NP, v + (uint64_t)((ks & 7) * 128), hi + (uint64_t)((ks & 7) * kStep + (ks >> 3) * (L::kP >> 4)), idesc_o, p.i > 0 || ks > 0);
        tc_commit(&bars.p_free[r % kB]);
        tc_commit(&bars.v_free[vr.slot]);
      }
      __syncwarp();
      vr.next(L::kV);
      leave(p);
      scores();
    }
  } else if (warp == 6) {
    // ------------------------------------------------------------ values that not every row sees
    bool ok = true;
    Ring vr;
    while (p.b < end) {
      enter(p);
      ok = wait(&bars.v_full[vr.slot], vr.pass);
      if (!__all_sync(0xffffffffu, ok)) break;
      const Share& g = p.g;
      const int j0 = block_key<kTcKeys>(g.all, g.blk0 + p.i);
      if (g.p_first < 0 || !seen_by_all(a, g.p_first, g.p_last, j0, j0 + kTcKeys - 1)) {
        const Seen own = paged_seen<kTcKeys>(a, g.p_first, g.p_last);
        const uint32_t block = values0 + vr.slot * L::kTile;
        bool bad = false;
        for (int row = lane; row < kTcKeys; row += 32) {
          const bool seen = seen_by_some(own, j0 + row);
          if (seen && g.p_first >= 0 && seen_by_all(a, g.p_first, g.p_last, j0 + row, j0 + row)) continue;
          for (int c = 0; c < D / 8; ++c) {
            const uint32_t at = block + (c / 8) * 16384 + row * 128 + (((c % 8) ^ (row & 7)) * 16);
            if (seen) {
              uint4 x;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
              bad = bad || not_finite2<T>(x.x) || not_finite2<T>(x.y) || not_finite2<T>(x.z) || not_finite2<T>(x.w);
            } else {
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0u) : "memory");
            }
          }
        }
        if (bad) s_bad = 1;
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.v_fixed[vr.slot]);
      vr.next(L::kV);
      leave(p);
    }
  } else if (warp < 4) {
    // ------------------------------------------------------------ weights: one key per thread
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const float scale = BIAS ? 1.0f : a.scale2;  // BIAS: scores are scaled when it is added
    constexpr float kLag = Num<T>::kLag, kLift = Num<T>::kLift;
    auto sync = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
    auto any = [](bool v) {
      int r;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((int)v) : "memory");
      return r != 0;
    };
    bool ok = true;
    float l[NP];
    for (int r = 0; p.b < end; ++r) {
      enter(p);
      const Share& g = p.g;
      const int j = block_key<kTcKeys>(g.all, g.blk0 + p.i) + tid, rows = g.ntok * a.group;
      const bool masked = g.p_first < 0 || !seen_by_all(a, g.p_first, g.p_last, j - tid, j - tid + kTcKeys - 1);
      const uint32_t s_col = tmem + (r & 1) * NP + lanes, o_col = tmem + 2 * NP + lanes;
      if (p.i == 0) {
#pragma unroll
        for (int c = 0; c < NP; ++c) l[c] = 0.0f;
        sync();  // (the last share's numbers have been read)
        if (tid < NP) s_ref[tid] = tid < rows ? -INFINITY : INFINITY, s_base2[tid] = tid < rows ? 0.0f : -INFINITY;  // (columns without a row: weights of 0)
        if (BIAS && tid < NP) s_far[tid] = tid < rows ? in_base2(a.bias[(size_t)(g.kvh * a.group + tid % a.group) * (a.bias_max + 1) + a.bias_max]) : 0.0f;
        sync();
      }
      ok = ok && all_wait(&bars.s_full[r & 1], (uint32_t)(r >> 1) & 1u);
      tc_fence_after();
      bool over = false;
      uint32_t v[kC];
      const bool near = BIAS && g.p_first - (j - tid + kTcKeys - 1) < a.bias_max;  // some distance has a bias of its own
      auto load = [&](int c0) {  // columns c0 .. c0 + kC - 1
        if constexpr (kC == 16) tmem_ld16(s_col + c0, v);
        else tmem_ld32(s_col + c0, v);
        tmem_ld_wait();
      };
      auto prepare = [&](int c0) {  // bias and mask
        if (BIAS) {
          if (near) {
            int tok = c0 / a.group, hg = c0 - tok * a.group;
#pragma unroll
            for (int i = 0; i < kC; ++i) {
              const float* table = a.bias + (size_t)(g.kvh * a.group + hg) * (a.bias_max + 1);
              const float b = c0 + i < rows ? in_base2(__ldg(table + max(0, min(g.p_first + tok - j, a.bias_max)))) : 0.0f;
              v[i] = __float_as_uint(fmaf(__uint_as_float(v[i]), a.scale2, b));
              if (++hg == a.group) hg = 0, ++tok;
            }
          } else {
#pragma unroll
            for (int i = 0; i < kC; ++i) v[i] = __float_as_uint(fmaf(__uint_as_float(v[i]), a.scale2, s_far[c0 + i]));
          }
        }
        if (masked) {
          int tok = c0 / a.group, hg = c0 - tok * a.group;
#pragma unroll
          for (int i = 0; i < kC; ++i) {
            if (!seen_by(a, g.p_first + tok, j)) v[i] = 0xff800000u;
            if (++hg == a.group) hg = 0, ++tok;
          }
        }
        if constexpr (NP > kC) {
          if (BIAS || masked) tmem_st32(s_col + c0, v);  // (they are read again)
        }
      };
#pragma unroll
      for (int c0 = 0; c0 < NP; c0 += kC) {
        load(c0);
        prepare(c0);
#pragma unroll
        for (int i = 0; i < kC; i += 4) {
          const float4 ref = *reinterpret_cast<const float4*>(s_ref + c0 + i);
          over |= fmaf(__uint_as_float(v[i]), scale, -kLag) > ref.x | fmaf(__uint_as_float(v[i + 1]), scale, -kLag) > ref.y |
                  fmaf(__uint_as_float(v[i + 2]), scale, -kLag) > ref.z | fmaf(__uint_as_float(v[i + 3]), scale, -kLag) > ref.w;
        }
      }
      if (NP > kC && (BIAS || masked)) tmem_st_wait();
      if (any(over)) {  // some row's maximum has outgrown its reference (always in an item's first block, unless nothing is seen)
#pragma unroll
        for (int c0 = 0; c0 < NP; c0 += kC) {
          if (NP > kC) load(c0);
#pragma unroll
          for (int i = 0; i < kC; ++i) {
            float x = __uint_as_float(v[i]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            if (lane == 0) s_max[warp][c0 + i] = x;
          }
        }
        sync();
        if (tid < rows) {
          const float old = s_ref[tid], top = fmaxf(fmaxf(s_max[0][tid], s_max[1][tid]), fmaxf(s_max[2][tid], s_max[3][tid])) * scale, now = fmaxf(old, top);
          s_alpha[tid] = now == -INFINITY ? 1.0f : exp2f(old - now);
          s_ref[tid] = now;
          s_base2[tid] = now == -INFINITY ? 0.0f : kLift - now;
        } else if (tid < NP) {
          s_alpha[tid] = 1.0f;
        }
        sync();
#pragma unroll
        for (int c = 0; c < NP; ++c) l[c] *= s_alpha[c];
        if (p.i > 0) {  // behind the products of the block before
          ok = ok && all_wait(&bars.p_free[(r - 1) % kB], (uint32_t)((r - 1) / kB) & 1u);
          tc_fence_after();
#pragma unroll
          for (int c0 = 0; c0 < NP; c0 += 16) {
            uint32_t o[16];
            tmem_ld16(o_col + c0, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * s_alpha[c0 + i]);
            tmem_st16(o_col + c0, o);
          }
          tmem_st_wait();
        }
      }
      if (r >= kB) ok = ok && all_wait(&bars.p_free[r % kB], (uint32_t)(r / kB - 1) & 1u);  // the products that read these weights' place
      const uint32_t row = p0 + r % kB * 2 * L::kP + tid * NP * 2;
#pragma unroll
      for (int c0 = 0; c0 < NP; c0 += kC) {
        if (NP > kC) load(c0);
#pragma unroll
        for (int c = 0; c < kC; c += 8) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = c + 2 * i;
            const float2 base = *reinterpret_cast<const float2*>(s_base2 + c0 + k);
            const float w0 = paged_exp2(fmaf(__uint_as_float(v[k]), scale, base.x)), w1 = paged_exp2(fmaf(__uint_as_float(v[k + 1]), scale, base.y));
            l[c0 + k] += w0, l[c0 + k + 1] += w1;
            hi[i] = Num<T>::pack(w0, w1);
            const float2 h = Num<T>::unpack(hi[i]);
            lo[i] = Num<T>::pack(w0 - h.x, w1 - h.y);
          }
          const int chunk = (c0 + c) / 8, sw = NP == 16 ? (tid >> 2) & 1 : NP == 32 ? (tid >> 1) & 3 : tid & 7;
          const uint32_t at = row + ((chunk ^ sw) * 16);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]) : "memory");
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + L::kP), "r"(lo[0]), "r"(lo[1]), "r"(lo[2]), "r"(lo[3]) : "memory");
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.p_ready[r & 1]);
      if (p.i == g.n - 1) {  // the share's end: the rows' sums, then a number of the value per thread
#pragma unroll
        for (int c = 0; c < NP; ++c) {
          float x = l[c];
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
          if (lane == 0) s_max[warp][c] = x;
        }
        sync();
        const size_t slot = (size_t)(2 * blockIdx.x + g.begins) * item_rows;
        if (tid < rows) {
          const int tok = tid / a.group, head = g.kvh * a.group + tid - tok * a.group;
          const float ref = s_ref[tid] - kLift, sink = g.whole && a.sink ? in_base2(a.sink[head]) : -INFINITY, most = fmaxf(ref, sink), at = most == -INFINITY ? 0.0f : most;
          const float f = exp2f(ref - at), sum = ((s_max[0][tid] + s_max[1][tid]) + (s_max[2][tid] + s_max[3][tid])) * f + exp2f(sink - at);
          s_alpha[tid] = !g.whole ? f : g.p_first + tok < 0 ? 0.0f : f / sum;
          if (!g.whole) w.part_ml[slot + tid] = make_float2(most, sum);
        }
        ok = ok && all_wait(&bars.p_free[r % kB], (uint32_t)(r / kB) & 1u);
        tc_fence_after();
        sync();
        if (tid < D && ok) {
          T* out = static_cast<T*>(a.out) + (long long)g.row0 * a.out_row + (long long)g.kvh * a.group * a.out_head + tid;
          float* part = w.part_o + slot * D + tid;
          int tok = 0, hg = 0;
          for (int c0 = 0; c0 < NP; c0 += 16) {
            uint32_t o[16];
            tmem_ld16(o_col + c0, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (c0 + i >= rows) break;
              const float x = g.p_first + tok < 0 ? 0.0f : __uint_as_float(o[i]) * s_alpha[c0 + i];
              if (g.whole) out[tok * a.out_row + hg * a.out_head] = T(x);
              else part[(size_t)(c0 + i) * D] = x;
              if (++hg == a.group) hg = 0, ++tok;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.o_free);
      }
      leave(p);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0) flags[blockIdx.x] = s_bad;
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kColumns);
  }
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static std::atomic<EncodeFn> fn{nullptr};
  EncodeFn f = fn.load(std::memory_order_acquire);
  if (!f) {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || !p) return nullptr;
    f = reinterpret_cast<EncodeFn>(p);
    fn.store(f, std::memory_order_release);
  }
  return f;
}
template <int N>
bool encode(CUtensorMap* map, CUtensorMapDataType type, const void* base, const cuuint64_t (&dims)[N], const cuuint64_t (&strides)[N - 1], const cuuint32_t (&box)[N]) {
  const EncodeFn fn = encode_fn();
  cuuint32_t one[N];
  for (auto& o : one) o = 1;
  return fn && fn(map, type, N, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int D, bool BIAS, bool EXACT>
cudaError_t configure() {
  static std::atomic<unsigned long long> done{0};
  return once_per_device(&done, [] { return cudaFuncSetAttribute(lm_paged_prompt_tc_kernel<T, D, BIAS, EXACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcLayout<D, BIAS>::kBytes); });
}
long long prompt_ctas(const Paged& a) {
  const int toks = 2 * (128 / a.group);
  return std::min((long long)a.rows, a.rows / toks + (long long)a.seqs) * a.kv_heads;
}
// CTAs that share a pair of tiles: as many as the GPU has room for, with four blocks of keys each at least.
int prompt_parts(const Paged& a) {
  const long long ctas = prompt_ctas(a), keys = std::min((long long)a.max_pages * a.page, a.window ? (long long)a.window + a.keep + 2 * (128 / a.group) : 1ll << 40);
  return ctas ? (int)std::max(1ll, std::min({16ll, kSms / ctas, keys / kTcKeys / 4})) : 1;
}
size_t prompt_split_rows(const Paged& a, int parts) { return (size_t)prompt_ctas(a) * parts * 256; }

template <class T, int D>
cudaError_t launch(const Paged& a, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, int piece, void* workspace, cudaStream_t s) {
  PromptSplit w{};
  w.parts = prompt_parts(a);
  if (w.parts > 1) {
    const size_t rows = prompt_split_rows(a, w.parts);
    w.part_o = static_cast<float*>(workspace);
    w.part_ml = reinterpret_cast<float2*>(w.part_o + rows * D);
    w.flags = reinterpret_cast<int*>(w.part_ml + rows);
  }
  const dim3 grid((unsigned)prompt_ctas(a), w.parts);
  auto go = [&](auto bias, auto exact) {
    constexpr bool BIAS = decltype(bias)::value, EXACT = decltype(exact)::value;
    const cudaError_t c = configure<T, D, BIAS, EXACT>();
    return c != cudaSuccess ? c : launch_pdl(lm_paged_prompt_tc_kernel<T, D, BIAS, EXACT>, grid, dim3(kTcThreads), TcLayout<D, BIAS>::kBytes, s, a, q, k, v, piece, w);
  };
  const std::true_type yes;
  const std::false_type no;
  const cudaError_t r = a.bias ? a.exact ? go(yes, yes) : go(yes, no) : a.exact ? go(no, yes) : go(no, no);
  return r != cudaSuccess || w.parts == 1 ? r : launch_pdl(lm_paged_prompt_join_kernel<T, D>, dim3(grid.x, 8), dim3(256), 0, s, a, w);
}

template <class T, int D, int NP, bool BIAS>
cudaError_t launch_decode_form(const Paged& a, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const DecodeWork& w, int* flags, int piece,
                               cudaStream_t s) {
  static std::atomic<unsigned long long> done{0};
  const auto kernel = lm_paged_decode_tc_kernel<T, D, NP, BIAS>;
  const cudaError_t r = once_per_device(&done, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DecLayout<D, NP>::kBytes); });
  if (r != cudaSuccess) return r;
  return launch_pdl(kernel, dim3(kDecCtas), dim3(kDecThreads), DecLayout<D, NP>::kBytes, s, a, q, k, v, w, flags, piece, paged_decode_tc_rows(a) / a.group);
}
template <class T, int D>
cudaError_t launch_decode(const Paged& a, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const DecodeWork& w, int* flags, int piece, cudaStream_t s) {
  const int rows = paged_decode_tc_rows(a);
  auto go = [&](auto np) {
    constexpr int NP = decltype(np)::value;
    return a.bias ? launch_decode_form<T, D, NP, true>(a, q, k, v, w, flags, piece, s) : launch_decode_form<T, D, NP, false>(a, q, k, v, w, flags, piece, s);
  };
  return rows <= 16 ? go(std::integral_constant<int, 16>()) : rows <= 32 ? go(std::integral_constant<int, 32>()) : go(std::integral_constant<int, 64>());
}

// Tensor maps of a call; false: addresses or strides that they do not take.
struct Maps {
  CUtensorMap q, k, v;
  int piece;
};
bool make_maps(const Paged& a, bool f16, int toks, Maps* m) {
  m->piece = 16;
  while (m->piece < kTcKeys && a.page % (2 * m->piece) == 0) m->piece *= 2;
  const auto type = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const cuuint32_t q_box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)toks}, box[4] = {64, (cuuint32_t)m->piece, 1, 1};
  const cuuint64_t D = a.dim, dims[4] = {D, (cuuint64_t)a.page, (cuuint64_t)a.kv_heads, (cuuint64_t)a.pages};
  return encode<3>(&m->q, type, a.q, {D, (cuuint64_t)a.heads, (cuuint64_t)a.rows}, {(cuuint64_t)a.q_head * 2, (cuuint64_t)a.q_row * 2}, q_box) &&
         encode<4>(&m->k, type, a.k, dims, {(cuuint64_t)a.k_row * 2, (cuuint64_t)a.k_head * 2, (cuuint64_t)a.k_page * 2}, box) &&
         encode<4>(&m->v, type, a.v, dims, {(cuuint64_t)a.v_row * 2, (cuuint64_t)a.v_head * 2, (cuuint64_t)a.v_page * 2}, box);
}

}  // namespace

bool prompt_tc_takes(const Paged& a) { return a.dim == a.vdim && (a.dim == 64 || a.dim == 128) && a.rows > 0 && prompt_ctas(a) <= 0x7fffffffll; }
size_t paged_prompt_bytes(const Paged& a) {
  if (!prompt_tc_takes(a)) return 0;
  const int parts = prompt_parts(a);
  return parts > 1 ? prompt_split_rows(a, parts) * (a.dim * 4 + sizeof(float2)) + (size_t)prompt_ctas(a) * parts * sizeof(int) : 0;
}
// Whether the kernel takes these sizes (and the tensor maps, these addresses and strides); `launched` says what became of it.
bool launch_paged_prompt_tc(const Paged& a, bool f16, void* workspace, cudaStream_t s, cudaError_t* launched) {
  if (!prompt_tc_takes(a) || !(a.scale2 > 1e-30f) || !(a.scale2 < 1e30f)) return false;
  const int toks = 128 / a.group;
  Maps m;
  if (!make_maps(a, f16, toks, &m)) return false;
  *launched = f16 ? (a.dim == 64 ? launch<__half, 64>(a, m.q, m.k, m.v, m.piece, workspace, s) : launch<__half, 128>(a, m.q, m.k, m.v, m.piece, workspace, s))
                  : (a.dim == 64 ? launch<__nv_bfloat16, 64>(a, m.q, m.k, m.v, m.piece, workspace, s) : launch<__nv_bfloat16, 128>(a, m.q, m.k, m.v, m.piece, workspace, s));
  return true;
}

bool paged_decode_tc_takes(const Paged& a) { return a.dim == a.vdim && (a.dim == 64 || a.dim == 128) && a.group <= 64; }
int paged_decode_tc_rows(const Paged& a) { return std::max(1, std::min(a.tokens, 64 / a.group)) * a.group; }
bool launch_paged_decode_tc(const Paged& a, bool f16, const DecodeWork& w, int* flags, cudaStream_t s, cudaError_t* launched) {
  if (!paged_decode_tc_takes(a) || !(a.scale2 > 1e-30f) || !(a.scale2 < 1e30f)) return false;
  if (((long long)a.max_pages * a.page / kTcKeys + 2) * a.seqs * a.kv_heads * w.row_blocks > 0x7fffffffll) return false;  // (blocks are counted in 32 bits)
  Maps m;
  if (!make_maps(a, f16, paged_decode_tc_rows(a) / a.group, &m)) return false;
  *launched = f16 ? (a.dim == 64 ? launch_decode<__half, 64>(a, m.q, m.k, m.v, w, flags, m.piece, s) : launch_decode<__half, 128>(a, m.q, m.k, m.v, w, flags, m.piece, s))
                  : (a.dim == 64 ? launch_decode<__nv_bfloat16, 64>(a, m.q, m.k, m.v, w, flags, m.piece, s)
                                 : launch_decode<__nv_bfloat16, 128>(a, m.q, m.k, m.v, w, flags, m.piece, s));
  return true;
}

}  // namespace lm
}  // namespace mllmb200
