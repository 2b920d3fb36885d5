// Attention with a gradient, head_dim 128, bf16 or fp16 operands on the tcgen05 tensor cores: the forward pass that also
// keeps the log-sum-exp of every row, and the backward pass, which recomputes the probabilities from it.
//
//   s_ij = c q_i.k_j   (c = softmax scale)      p_ij = exp(s_ij - lse_i)      o_i = sum_j p_ij v_j
//   D_i = do_i.o_i     dp_ij = do_i.v_j         ds_ij = p_ij (dp_ij - D_i)
//   dq_i = c sum_j ds_ij k_j      dk_j = c sum_i ds_ij q_i      dv_j = sum_i p_ij do_i
//
// The backward pass is TWO kernels, one that owns query rows (dq) and one that owns key rows (dk and dv), each with its
// sums in tensor memory from the first product to the last.  One kernel for all three would do five products per tile
// instead of seven, but its dq would have to leave the SM as fp32 atomics for every tile (64 KB per pair of tiles, an
// order of addition that changes from run to run) and, with a 128-wide tile of one SM, its operand reads need more
// shared-memory bandwidth than the seven products here, four of which take their A operand from tensor memory.
//
// q_lens / k_lens (per sample, optional) bound the tokens that exist: rows behind a length take no part in anything (not
// even when they hold NaN or infinity), their outputs are zero and their lse is -inf, and so are those of queries that
// see no key at all.
//
// Scores, probabilities, row statistics, D and all sums are fp32.  p and ds are rounded once to the operands' type, as A
// operands of the second products (the tensor cores take nothing wider together with 16-bit B operands).
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace dax {
namespace {

constexpr int BOX_BYTES = 128 * 128;       // one [128 rows x 64 channels] box
constexpr int TILE_BYTES = 2 * BOX_BYTES;  // a [128 x 128] tile of 16-bit elements
constexpr int THREADS = 384;
constexpr int PRODUCER_WARP = 8, ISSUER_WARP0 = 9, ISSUER_WARP1 = 10, TMEM_WARP = 11;
constexpr float TAU = 8.f;                 // forward: lazy rescale, p <= 2^8
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int kMaxSplits = 16;

struct Rows { const void* p; int64_t sb, sh, st; };  // a [B, heads, S, 128] view: element strides of sample, head, token

struct TrainParams {
  Rows q, k, v, o, dout, dq, dk, dv;
  float* lse;          // [BH, Sq]
  const int* q_lens;   // [B] or null
  const int* k_lens;
  float* row_stats;    // backward: [BH, Sq_pad, ...] as [2][BH * Sq_pad]: lse * log2(e) (+inf: no such row), then D
  float* part;         // split runs: fp32 partial sums
  float* part_lse;     // split forward runs: [splits, BH, Sq] row maxima-free log2 sums
  int* status;
  int B, heads, Sq, Sk, Sq_pad, splits;
  float sm_scale;
};

__device__ __forceinline__ void reg_alloc_216() { asm volatile("setmaxnreg.inc.sync.aligned.u32 216;"); }
__device__ __forceinline__ void reg_dealloc_72() { asm volatile("setmaxnreg.dec.sync.aligned.u32 72;"); }

template <bool BF16>
__device__ __forceinline__ uint32_t pack_rn(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool BF16>
__device__ __forceinline__ void unpack(uint32_t w, float& lo, float& hi) {
  if constexpr (BF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  }
}
__device__ __forceinline__ int valid_len(const int* lens, int b, int S) { return lens != nullptr ? min(max(lens[b], 0), S) : S; }

__device__ __forceinline__ const uint16_t* row_ptr(const Rows& t, int b, int h, int64_t s) {
  return static_cast<const uint16_t*>(t.p) + b * t.sb + h * t.sh + s * t.st;
}
__device__ __forceinline__ uint16_t* out_ptr(const Rows& t, int b, int h, int64_t s) { return const_cast<uint16_t*>(row_ptr(t, b, h, s)); }

// 32 fp32 values -> 64 bytes of 16-bit results
template <bool BF16>
__device__ __forceinline__ void store_row32(uint16_t* dst, const uint32_t (&v)[32], float mul) {
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = pack_rn<BF16>(__uint_as_float(v[i + 2 * k]) * mul, __uint_as_float(v[i + 2 * k + 1]) * mul);
    *reinterpret_cast<uint4*>(dst + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
__device__ __forceinline__ void store_zero(uint16_t* dst, int elements) {
  for (int i = 0; i < elements; i += 8) *reinterpret_cast<uint4*>(dst + i) = make_uint4(0u, 0u, 0u, 0u);
}

// ---- ring of tiles --------------------------------------------------------------------------------------------------
struct TileLoad {
  uint8_t* dst;
  const CUtensorMap* map;
  int row, h, b;
};
__device__ __forceinline__ void issue_tile(const TileLoad& t, uint64_t* bar) {
#pragma unroll
  for (int sub = 0; sub < 2; ++sub) tma_load_4d(t.dst + sub * BOX_BYTES, t.map, bar, sub * 64, t.row, t.h, t.b);
}
// A tile whose rows from `rem` on lie behind the sequence's length, but inside the tensor, may hold anything, and a zero
// probability does not silence a NaN in a product.  The tile is fetched on a barrier of its own (phase `ph`), those rows
// are overwritten with zeros, and only then does the ring slot become full.  Called by the whole producer warp.
__device__ __forceinline__ bool load_tile_tail(const TileLoad& t, uint64_t* tail_bar, uint32_t ph, int rem, uint64_t* full,
                                               volatile uint32_t* abort_flag) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) {
    mbar_arrive_expect_tx(tail_bar, TILE_BYTES);
    issue_tile(t, tail_bar);
  }
  __syncwarp();
  if (!mbar_wait(tail_bar, ph, abort_flag)) return false;
  for (int sub = 0; sub < 2; ++sub)
    for (int i = rem * 8 + lane; i < 128 * 8; i += 32)
      *reinterpret_cast<uint4*>(t.dst + sub * BOX_BYTES + i * 16) = make_uint4(0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) mbar_arrive(full);
  return true;
}

// A[smem, K-major] . B[smem, K-major]^T over 128 channels: 8 steps of 16, box `i / 4` holds channels [64 (i / 4), +64)
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_smem, uint32_t b_smem, uint32_t idesc) {
  const uint64_t a = make_desc_k_sw128(a_smem), b = make_desc_k_sw128(b_smem);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint64_t adv = static_cast<uint64_t>((i >> 2) * (BOX_BYTES >> 4) + 2 * (i & 3));
    umma_ss<KIND_F16>(d, a + adv, b + adv, idesc, i != 0 ? 1u : 0u);
  }
}
// the same with A in tensor memory (64 columns, two elements each)
__device__ __forceinline__ void mma_ts_k(uint32_t d, uint32_t a_tmem, uint32_t b_smem, uint32_t idesc) {
  const uint64_t b = make_desc_k_sw128(b_smem);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint64_t adv = static_cast<uint64_t>((i >> 2) * (BOX_BYTES >> 4) + 2 * (i & 3));
    umma_ts_f16(d, a_tmem + 8 * i, b + adv, idesc, i != 0 ? 1u : 0u);
  }
}
// D += A[tmem] . B[smem] with the contraction over the tile's rows: B is MN-major, 16 rows per step.  The second four
// steps take A from `a_hi` columns further.
__device__ __forceinline__ void mma_ts_mn(uint32_t d, uint32_t a_tmem, uint32_t a_hi, uint32_t b_smem, uint32_t idesc, bool first) {
  const uint64_t b = make_desc_mn_sw128(b_smem, BOX_BYTES);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    umma_ts_f16(d, a_tmem + (i >= 4 ? a_hi : 0u) + 8 * (i & 3), b + static_cast<uint64_t>(i * ((16 * 128) >> 4)), idesc,
                (!first || i != 0) ? 1u : 0u);
}
template <bool BF16>
__device__ __forceinline__ uint32_t idesc_k() { return make_idesc(1, BF16 ? 1 : 0, BF16 ? 1 : 0, 128, 128); }
template <bool BF16>
__device__ __forceinline__ uint32_t idesc_mn() { return idesc_k<BF16>() | (1u << 16); }  // B is MN-major

// Set-up and tear-down shared by the kernels
__device__ __forceinline__ uint32_t open_tmem(uint32_t* slot, int warp) {
  if (warp == TMEM_WARP) {
    tmem_alloc(slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  return *slot;
}
__device__ __forceinline__ void close_tmem(uint32_t base, int warp, volatile uint32_t* abort_flag, int* status) {
  tc_fence_before_sync();
  __syncthreads();
  if (warp == TMEM_WARP) {
    tc_fence_after_sync();
    tmem_dealloc(base, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) atomicExch(status, DAX_ERR_TIMEOUT);
}

// ---- dq ----------------------------------------------------------------------------------------------------------------
// One CTA = 128 query rows of one head.  q and do of these rows are the A operands of the first two products for every
// tile of keys, so they live in TENSOR memory, as does ds: every product takes A from there and only k and v tiles pass
// through shared memory.
//   warps 0..7   one thread = one query row x 64 keys of the tile (warps 0-3: the first 64)
//   warp  8      TMA producer: k_0, v_0, k_1, ... through the ring
//   warp  9      issues s = q.k_j^T        warp 10  issues dp = do.v_j^T and dq += ds.k_j
// Tensor memory: s [0,128)  dp [128,256), ds over the first half of each thread's own columns of it  dq [256,384)
// q [384,448)  do [448,512).  s is free as soon as it is in registers, so s of the next tile is computed under ds of this
// one, and dp of the next tile under its exponentials.
constexpr int DQ_SLOTS = 6;
constexpr int DQ_OFF_STAT = DQ_SLOTS * TILE_BYTES;
constexpr int DQ_OFF_BAR = DQ_OFF_STAT + 1024;
constexpr int DQ_SMEM = DQ_OFF_BAR + 256 + 1024;

template <bool BF16>
__global__ void __launch_bounds__(THREADS, 1)
attn_bwd_dq_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TrainParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q0 = blockIdx.x * 128, bh = blockIdx.y, b = bh / p.heads, h = bh % p.heads, split = blockIdx.z;
  const int q_len = valid_len(p.q_lens, b, p.Sq), k_len = valid_len(p.k_lens, b, p.Sk);
  const int n_all = q0 < q_len ? (k_len + 127) / 128 : 0;
  const int per = (n_all + p.splits - 1) / p.splits;
  const int j0 = split * per, n = max(0, min(n_all, j0 + per) - j0);
  const int r = (warp & 3) * 32 + lane, half = (warp >> 2) & 1, q_row = q0 + r;
  // a split run leaves fp32 sums [split][BH][Sq][128] that are joined afterwards
  float* part = p.part + ((static_cast<int64_t>(split) * p.B * p.heads + bh) * p.Sq + q_row) * 128 + half * 64;
  const int64_t stat = static_cast<int64_t>(bh) * p.Sq_pad + q_row;
  const int64_t stats = static_cast<int64_t>(p.B) * p.heads * p.Sq_pad;

  if (n == 0) {  // nothing to see: zeros
    if (warp < 8) {
      if (half == 0 && split == 0) {
        p.row_stats[stat] = INFINITY;
        p.row_stats[stats + stat] = 0.f;
      }
      if (q_row < p.Sq) {
        if (p.splits > 1) {
          for (int i = 0; i < 64; i += 4) *reinterpret_cast<float4*>(part + i) = make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
          store_zero(out_ptr(p.dq, b, h, q_row) + half * 64, 64);
        }
      }
    }
    return;
  }

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + DQ_OFF_BAR);
  uint64_t* full = bars;                 // [DQ_SLOTS]
  uint64_t* empty = full + DQ_SLOTS;     // [DQ_SLOTS]
  uint64_t* tail = empty + DQ_SLOTS;
  uint64_t* a_full = tail + 1;           // q and do are in tensor memory
  uint64_t* s_full = a_full + 1;
  uint64_t* s_free = s_full + 1;
  uint64_t* dp_full = s_free + 1;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* dq_done = ds_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dq_done + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < DQ_SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(tail, 1);
    mbar_init(a_full, 8);
    mbar_init(s_full, 1);
    mbar_init(s_free, 8);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 8);
    mbar_init(dq_done, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  const uint32_t tm = open_tmem(tmem_slot, warp);
  constexpr uint32_t T_S = 0, T_DP = 128, T_DQ = 256, T_Q = 384, T_DO = 448;

  if (warp >= PRODUCER_WARP) {
    reg_dealloc_72();
    if (warp == PRODUCER_WARP) {
      const int rem = k_len < p.Sk ? k_len % 128 : 0;  // rows of the last tile of k that exist (0: no tail to clear)
      for (int seq = 0; seq < 2 * n; ++seq) {
        const int j = j0 + (seq >> 1);
        const uint32_t s = seq % DQ_SLOTS, ph = (seq / DQ_SLOTS) & 1u;
        if (!mbar_wait(&empty[s], ph ^ 1u, abort_flag)) break;
        const TileLoad t = {smem + s * TILE_BYTES, (seq & 1) ? &map_v : &map_k, j * 128, h, b};
        if (rem != 0 && j == n_all - 1 && (seq & 1) == 0) {
          if (!load_tile_tail(t, tail, 0, rem, &full[s], abort_flag)) break;
        } else if (lane == 0) {
          mbar_arrive_expect_tx(&full[s], TILE_BYTES);
          issue_tile(t, &full[s]);
        }
        __syncwarp();
      }
    } else if (warp == ISSUER_WARP0) {
      const bool leader = elect_one();
      const uint32_t ring = smem_u32(smem), id = idesc_k<BF16>();
      bool ok = mbar_wait(a_full, 0, abort_flag);
      for (int j = 0; ok && j < n; ++j) {
        const uint32_t seq = 2 * j, s = seq % DQ_SLOTS, ph = (seq / DQ_SLOTS) & 1u;
        ok = mbar_wait(&full[s], ph, abort_flag) && (j == 0 || mbar_wait(s_free, (j - 1) & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          mma_ts_k(tm + T_S, tm + T_Q, ring + s * TILE_BYTES, id);
          umma_commit(s_full);
        }
        __syncwarp();
      }
    } else if (warp == ISSUER_WARP1) {
      const bool leader = elect_one();
      const uint32_t ring = smem_u32(smem), id = idesc_k<BF16>(), id_mn = idesc_mn<BF16>();
      bool ok = mbar_wait(a_full, 0, abort_flag);
      for (int j = 0; ok && j < n; ++j) {
        const uint32_t seq = 2 * j + 1, s = seq % DQ_SLOTS, ph = (seq / DQ_SLOTS) & 1u;
        // dp lies where ds of the last tile was read: that product has to be over
        ok = mbar_wait(&full[s], ph, abort_flag) && (j == 0 || mbar_wait(dq_done, (j - 1) & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          mma_ts_k(tm + T_DP, tm + T_DO, ring + s * TILE_BYTES, id);
          umma_commit(dp_full);
          umma_commit(&empty[s]);
        }
        __syncwarp();
        ok = mbar_wait(ds_full, j & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t ks = (2 * j) % DQ_SLOTS;
        if (leader) {
          mma_ts_mn(tm + T_DQ, tm + T_DP, 64, ring + ks * TILE_BYTES, id_mn, j == 0);
          umma_commit(dq_done);
          umma_commit(&empty[ks]);
        }
        __syncwarp();
      }
    }
  } else {
    reg_alloc_216();
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const bool live = q_row < q_len;
    float* s_stat = reinterpret_cast<float*>(smem + DQ_OFF_STAT);  // [2][128]: lse * log2 e, D
    // warps 0-3 bring q, warps 4-7 bring do and compute D
    {
      uint32_t w[32];
      const Rows& src = half == 0 ? p.q : p.dout;
      float d = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          uint4 u = make_uint4(0u, 0u, 0u, 0u);
          if (live) u = *reinterpret_cast<const uint4*>(row_ptr(src, b, h, q_row) + c * 64 + 2 * i);
          w[i] = u.x; w[i + 1] = u.y; w[i + 2] = u.z; w[i + 3] = u.w;
        }
        tmem_st32(tm + lanes + (half == 0 ? T_Q : T_DO) + 32 * c, w);
        if (half == 1 && live) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(row_ptr(p.o, b, h, q_row) + c * 64 + 2 * i);
            const uint32_t ow[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float a0, a1, o0, o1;
              unpack<BF16>(w[i + k], a0, a1);
              unpack<BF16>(ow[k], o0, o1);
              d = fmaf(a0, o0, d);
              d = fmaf(a1, o1, d);
            }
          }
        }
      }
      tmem_wait_st();
      tc_fence_before_sync();
      if (half == 1) {
        float l2 = INFINITY;
        if (live) {
          const float l = p.lse[static_cast<int64_t>(bh) * p.Sq + q_row];
          l2 = l == -INFINITY ? INFINITY : l * LOG2E;
        }
        s_stat[r] = l2;
        s_stat[128 + r] = d;
        if (split == 0) {
          p.row_stats[stat] = l2;
          p.row_stats[stats + stat] = d;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(a_full);
    }
    bool ok = mbar_wait(a_full, 0, abort_flag);  // all 8 warps have arrived: s_stat is complete
    const float neg_l2 = -s_stat[r], neg_d = -s_stat[128 + r];
    const float cmul = p.sm_scale * LOG2E;
    for (int j = 0; ok && j < n; ++j) {
      const int valid = k_len - (j0 + j) * 128 - half * 64;  // this thread's columns that exist
      if (!(ok = mbar_wait(s_full, j & 1u, abort_flag))) break;
      tc_fence_after_sync();
      uint32_t sv[64];
      tmem_ld32(tm + lanes + T_S + half * 64, *reinterpret_cast<uint32_t(*)[32]>(&sv[0]));
      tmem_ld32(tm + lanes + T_S + half * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(&sv[32]));
      tmem_wait_ld();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free);
#pragma unroll
      for (int i = 0; i < 64; ++i) sv[i] = __float_as_uint(ex2(fmaf(__uint_as_float(sv[i]), cmul, neg_l2)));
      if (!(ok = mbar_wait(dp_full, j & 1u, abort_flag))) break;
      tc_fence_after_sync();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t dp[32];
        tmem_ld32(tm + lanes + T_DP + half * 64 + 32 * c, dp);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i)
          sv[32 * c + i] = __float_as_uint(__uint_as_float(sv[32 * c + i]) * (__uint_as_float(dp[i]) + neg_d));
      }
      if (valid < 64) {  // keys behind the length: whatever their scores were
#pragma unroll
        for (int i = 0; i < 64; ++i) sv[i] = i < valid ? sv[i] : 0u;
      }
      uint32_t pk[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) pk[i] = pack_rn<BF16>(__uint_as_float(sv[2 * i]), __uint_as_float(sv[2 * i + 1]));
      tmem_st32(tm + lanes + T_DP + half * 64, pk);
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    if (ok && mbar_wait(dq_done, (n - 1) & 1u, abort_flag)) {
      tc_fence_after_sync();
      // the softmax over one key is constant: its gradient is zero, not the rounding of dp - D
      const float mul = k_len == 1 ? 0.f : p.sm_scale;
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        uint32_t v[32];
        tmem_ld32(tm + lanes + T_DQ + half * 64 + 32 * c, v);
        tmem_wait_ld();
        if (q_row >= p.Sq) continue;
        if (p.splits > 1) {
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(part + 32 * c + i) = live ? make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]) : make_uint4(0u, 0u, 0u, 0u);
        } else if (live) {
          store_row32<BF16>(out_ptr(p.dq, b, h, q_row) + half * 64 + 32 * c, v, mul);
        } else {
          store_zero(out_ptr(p.dq, b, h, q_row) + half * 64 + 32 * c, 32);
        }
      }
    }
  }
  close_tmem(tm, warp, abort_flag, p.status);
}

// ---- dk, dv ------------------------------------------------------------------------------------------------------------
// One CTA = 128 keys of one head; k and v stay in shared memory, q and do tiles pass through the ring.  Everything is
// transposed: a thread owns a KEY row x 64 queries, so p^T and ds^T come out as A operands of dv += p^T.do and
// dk += ds^T.q and never leave tensor memory; lse and D of the queries are read along the row.
//   warp 9   issues s^T = k.q_i^T and dv += p^T.do_i        warp 10  issues dp^T = v.do_i^T and dk += ds^T.q_i
// Tensor memory: s^T [0,128), p^T over it   dp^T [128,256), ds^T over it   dv [256,384)   dk [384,512).
constexpr int KV_SLOTS = 4;
constexpr int KV_OFF_K = KV_SLOTS * TILE_BYTES;
constexpr int KV_OFF_V = KV_OFF_K + TILE_BYTES;
constexpr int KV_OFF_STAT = KV_OFF_V + TILE_BYTES;  // [2 stages][2][128] floats
constexpr int KV_OFF_BAR = KV_OFF_STAT + 2048;
constexpr int KV_SMEM = KV_OFF_BAR + 256 + 1024;

template <bool BF16>
__global__ void __launch_bounds__(THREADS, 1)
attn_bwd_dkdv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                     const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TrainParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k0 = blockIdx.x * 128, bh = blockIdx.y, b = bh / p.heads, h = bh % p.heads, split = blockIdx.z;
  const int q_len = valid_len(p.q_lens, b, p.Sq), k_len = valid_len(p.k_lens, b, p.Sk);
  const int n_all = k0 < k_len ? (q_len + 127) / 128 : 0;
  const int per = (n_all + p.splits - 1) / p.splits;
  const int i0 = split * per, n = max(0, min(n_all, i0 + per) - i0);
  const int r = (warp & 3) * 32 + lane, half = (warp >> 2) & 1, k_row = k0 + r;
  // a split run leaves fp32 sums: dk [split][BH][Sk][128], then dv the same
  const int64_t part_all = static_cast<int64_t>(p.splits) * p.B * p.heads * p.Sk * 128;
  float* part = p.part + ((static_cast<int64_t>(split) * p.B * p.heads + bh) * p.Sk + k_row) * 128 + half * 64;

  if (n == 0) {
    if (warp < 8 && k_row < p.Sk) {
      if (p.splits > 1) {
        for (int i = 0; i < 64; i += 4) {
          *reinterpret_cast<float4*>(part + i) = make_float4(0.f, 0.f, 0.f, 0.f);
          *reinterpret_cast<float4*>(part + part_all + i) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
      } else {
        store_zero(out_ptr(p.dk, b, h, k_row) + half * 64, 64);
        store_zero(out_ptr(p.dv, b, h, k_row) + half * 64, 64);
      }
    }
    return;
  }

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + KV_OFF_BAR);
  uint64_t* full = bars;                // [KV_SLOTS]
  uint64_t* empty = full + KV_SLOTS;    // [KV_SLOTS] released by the two products that read the tile
  uint64_t* tail = empty + KV_SLOTS;
  uint64_t* kv_full = tail + 1;
  uint64_t* s_full = kv_full + 1;
  uint64_t* p_full = s_full + 1;
  uint64_t* dv_done = p_full + 1;
  uint64_t* dp_full = dv_done + 1;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* dk_done = ds_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dk_done + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < KV_SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 2);
    }
    mbar_init(tail, 1);
    mbar_init(kv_full, 1);
    mbar_init(s_full, 1);
    mbar_init(p_full, 8);
    mbar_init(dv_done, 1);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 8);
    mbar_init(dk_done, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  const uint32_t tm = open_tmem(tmem_slot, warp);
  constexpr uint32_t T_S = 0, T_DP = 128, T_DV = 256, T_DK = 384;
  const int64_t stats = static_cast<int64_t>(p.B) * p.heads * p.Sq_pad;

  if (warp >= PRODUCER_WARP) {
    reg_dealloc_72();
    if (warp == PRODUCER_WARP) {
      if (lane == 0) {
        mbar_arrive_expect_tx(kv_full, 2 * TILE_BYTES);
        issue_tile({smem + KV_OFF_K, &map_k, k0, h, b}, kv_full);
        issue_tile({smem + KV_OFF_V, &map_v, k0, h, b}, kv_full);
      }
      __syncwarp();
      const int rem = q_len < p.Sq ? q_len % 128 : 0;
      for (int seq = 0; seq < 2 * n; ++seq) {
        const int i = i0 + (seq >> 1);
        const uint32_t s = seq % KV_SLOTS, ph = (seq / KV_SLOTS) & 1u;
        if (!mbar_wait(&empty[s], ph ^ 1u, abort_flag)) break;
        const bool is_q = (seq & 1) == 0, clear = rem != 0 && i == n_all - 1;
        const TileLoad t = {smem + s * TILE_BYTES, is_q ? &map_q : &map_do, i * 128, h, b};
        if (lane == 0) {
          // lse and D of the tile's queries ride on the q tile's barrier; the stage is free with the slot
          const uint32_t bytes = (is_q ? 1024 : 0) + (clear ? 0 : TILE_BYTES);
          if (bytes != 0 && !clear) mbar_arrive_expect_tx(&full[s], bytes);
          if (is_q) {
            float* dst = reinterpret_cast<float*>(smem + KV_OFF_STAT) + (seq / 2 % 2) * 256;
            const float* src = p.row_stats + static_cast<int64_t>(bh) * p.Sq_pad + i * 128;
            if (clear) {  // the arrival comes from load_tile_tail
              asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full[s])), "r"(1024u) : "memory");
            }
            bulk_load(dst, src, 512, &full[s]);
            bulk_load(dst + 128, src + stats, 512, &full[s]);
          }
          if (!clear) issue_tile(t, &full[s]);
        }
        __syncwarp();
        if (clear && !load_tile_tail(t, tail, is_q ? 0u : 1u, rem, &full[s], abort_flag)) break;
      }
    } else if (warp == ISSUER_WARP0) {
      const bool leader = elect_one();
      const uint32_t ring = smem_u32(smem), id = idesc_k<BF16>(), id_mn = idesc_mn<BF16>();
      bool ok = mbar_wait(kv_full, 0, abort_flag);
      for (int i = 0; ok && i < n; ++i) {
        const uint32_t seq = 2 * i, s = seq % KV_SLOTS, ph = (seq / KV_SLOTS) & 1u, s1 = (seq + 1) % KV_SLOTS, ph1 = ((seq + 1) / KV_SLOTS) & 1u;
        // s^T lies where p^T of the last tile was read: that product has to be over
        ok = mbar_wait(&full[s], ph, abort_flag) && (i == 0 || mbar_wait(dv_done, (i - 1) & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          mma_ss(tm + T_S, ring + KV_OFF_K, ring + s * TILE_BYTES, id);
          umma_commit(s_full);
          umma_commit(&empty[s]);
        }
        __syncwarp();
        ok = mbar_wait(&full[s1], ph1, abort_flag) && mbar_wait(p_full, i & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          mma_ts_mn(tm + T_DV, tm + T_S, 64, ring + s1 * TILE_BYTES, id_mn, i == 0);
          umma_commit(dv_done);
          umma_commit(&empty[s1]);
        }
        __syncwarp();
      }
    } else if (warp == ISSUER_WARP1) {
      const bool leader = elect_one();
      const uint32_t ring = smem_u32(smem), id = idesc_k<BF16>(), id_mn = idesc_mn<BF16>();
      bool ok = mbar_wait(kv_full, 0, abort_flag);
      for (int i = 0; ok && i < n; ++i) {
        const uint32_t seq = 2 * i, s = seq % KV_SLOTS, ph = (seq / KV_SLOTS) & 1u, s1 = (seq + 1) % KV_SLOTS, ph1 = ((seq + 1) / KV_SLOTS) & 1u;
        ok = mbar_wait(&full[s1], ph1, abort_flag) && (i == 0 || mbar_wait(dk_done, (i - 1) & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          mma_ss(tm + T_DP, ring + KV_OFF_V, ring + s1 * TILE_BYTES, id);
          umma_commit(dp_full);
          umma_commit(&empty[s1]);
        }
        __syncwarp();
        ok = mbar_wait(&full[s], ph, abort_flag) && mbar_wait(ds_full, i & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          mma_ts_mn(tm + T_DK, tm + T_DP, 64, ring + s * TILE_BYTES, id_mn, i == 0);
          umma_commit(dk_done);
          umma_commit(&empty[s]);
        }
        __syncwarp();
      }
    }
  } else {
    reg_alloc_216();
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const float cmul = p.sm_scale * LOG2E;
    bool ok = true;
    for (int i = 0; ok && i < n; ++i) {
      const float* stat = reinterpret_cast<const float*>(smem + KV_OFF_STAT) + (i % 2) * 256 + half * 64;
      const uint32_t seq = 2 * i;
      ok = mbar_wait(&full[seq % KV_SLOTS], (seq / KV_SLOTS) & 1u, abort_flag) && mbar_wait(s_full, i & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after_sync();
      uint32_t sv[64];
      tmem_ld32(tm + lanes + T_S + half * 64, *reinterpret_cast<uint32_t(*)[32]>(&sv[0]));
      tmem_ld32(tm + lanes + T_S + half * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(&sv[32]));
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        const float4 l2 = *reinterpret_cast<const float4*>(stat + c);
        sv[c] = __float_as_uint(ex2(fmaf(__uint_as_float(sv[c]), cmul, -l2.x)));
        sv[c + 1] = __float_as_uint(ex2(fmaf(__uint_as_float(sv[c + 1]), cmul, -l2.y)));
        sv[c + 2] = __float_as_uint(ex2(fmaf(__uint_as_float(sv[c + 2]), cmul, -l2.z)));
        sv[c + 3] = __float_as_uint(ex2(fmaf(__uint_as_float(sv[c + 3]), cmul, -l2.w)));
      }
      {
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) pk[c] = pack_rn<BF16>(__uint_as_float(sv[2 * c]), __uint_as_float(sv[2 * c + 1]));
        tmem_st32(tm + lanes + T_S + half * 64, pk);
      }
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
      if (!(ok = mbar_wait(dp_full, i & 1u, abort_flag))) break;
      tc_fence_after_sync();
      uint32_t pk[32];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t dp[32];
        tmem_ld32(tm + lanes + T_DP + half * 64 + 32 * c, dp);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 d = *reinterpret_cast<const float4*>(stat + 128 + 32 * c + k);
          const float e0 = __uint_as_float(sv[32 * c + k]) * (__uint_as_float(dp[k]) - d.x);
          const float e1 = __uint_as_float(sv[32 * c + k + 1]) * (__uint_as_float(dp[k + 1]) - d.y);
          const float e2 = __uint_as_float(sv[32 * c + k + 2]) * (__uint_as_float(dp[k + 2]) - d.z);
          const float e3 = __uint_as_float(sv[32 * c + k + 3]) * (__uint_as_float(dp[k + 3]) - d.w);
          pk[16 * c + k / 2] = pack_rn<BF16>(e0, e1);
          pk[16 * c + k / 2 + 1] = pack_rn<BF16>(e2, e3);
        }
      }
      tmem_st32(tm + lanes + T_DP + half * 64, pk);
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    if (ok && mbar_wait(dv_done, (n - 1) & 1u, abort_flag) && mbar_wait(dk_done, (n - 1) & 1u, abort_flag)) {
      tc_fence_after_sync();
      const bool live = k_row < k_len;
      const float mul = k_len == 1 ? 0.f : p.sm_scale;  // one key: see the dq kernel
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        const bool is_k = c < 2;
        const int at = (c & 1) * 32;
        uint32_t v[32];
        tmem_ld32(tm + lanes + (is_k ? T_DK : T_DV) + half * 64 + at, v);
        tmem_wait_ld();
        if (k_row >= p.Sk) continue;
        if (p.splits > 1) {
          float* dst = part + (is_k ? 0 : part_all) + at;
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(dst + i) = live ? make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]) : make_uint4(0u, 0u, 0u, 0u);
        } else {
          uint16_t* dst = out_ptr(is_k ? p.dk : p.dv, b, h, k_row) + half * 64 + at;
          if (live) store_row32<BF16>(dst, v, is_k ? mul : 1.f);
          else store_zero(dst, 32);
        }
      }
    }
  }
  close_tmem(tm, warp, abort_flag, p.status);
}

// ---- forward -----------------------------------------------------------------------------------------------------------
// The schedule of attn_fwd_tmem_p_kernel (attn_tmem.cu: 256 query rows per CTA as two tiles, one shared score buffer,
// probabilities through tensor memory, five-slot ring of k and v tiles) with what training asks of it: lengths, fp16,
// any strides, the log-sum-exp, probabilities rounded instead of truncated, and, where there are too few rows to fill the
// GPU, the keys split over several CTAs.
constexpr int F_SLOTS = 5;
constexpr int F_OFF_Q = 0;
constexpr int F_OFF_RING = 2 * TILE_BYTES;
constexpr int F_OFF_BAR = F_OFF_RING + F_SLOTS * TILE_BYTES;
constexpr int F_SMEM = F_OFF_BAR + 256 + 1024;

template <bool BF16>
__global__ void __launch_bounds__(THREADS, 1)
attn_fwd_lse_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const TrainParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q0 = blockIdx.x * 256, bh = blockIdx.y, b = bh / p.heads, h = bh % p.heads, split = blockIdx.z;
  const int q_len = valid_len(p.q_lens, b, p.Sq), k_len = valid_len(p.k_lens, b, p.Sk);
  const int n_all = q0 < q_len ? (k_len + 127) / 128 : 0;
  const int per = (n_all + p.splits - 1) / p.splits;
  const int j0 = split * per, n = max(0, min(n_all, j0 + per) - j0);
  const int tiles = q0 + 128 < q_len ? 2 : 1;  // the second tile may have no rows at all
  const int x = warp >> 2, r = (warp & 3) * 32 + lane, q_row = q0 + x * 128 + r;
  const int64_t row = static_cast<int64_t>(bh) * p.Sq + q_row;
  const int64_t split_row = static_cast<int64_t>(split) * p.B * p.heads * p.Sq + row;
  auto store_nothing = [&]() {
    if (q_row >= p.Sq) return;
    if (p.splits > 1) {  // a part without keys: zero weight
      p.part_lse[split_row] = -INFINITY;
      for (int i = 0; i < 128; i += 4) *reinterpret_cast<float4*>(p.part + split_row * 128 + i) = make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
      p.lse[row] = -INFINITY;
      store_zero(out_ptr(p.o, b, h, q_row), 128);
    }
  };
  if (n == 0) {
    if (warp < 8) store_nothing();
    return;
  }

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + F_OFF_BAR);
  uint64_t* q_full = bars;
  uint64_t* kv_full = bars + 1;            // [F_SLOTS]
  uint64_t* kv_empty = kv_full + F_SLOTS;  // [F_SLOTS] released by one product per query tile
  uint64_t* tail = kv_empty + F_SLOTS;
  uint64_t* s_full = tail + 1;             // [2]
  uint64_t* s_free = s_full + 2;
  uint64_t* p_full = s_free + 1;           // [2]
  uint64_t* pv_done = p_full + 2;          // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(tail, 1);
    for (int i = 0; i < F_SLOTS; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], tiles);
    }
    mbar_init(s_free, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  const uint32_t tm = open_tmem(tmem_slot, warp);

  if (warp >= PRODUCER_WARP) {
    reg_dealloc_72();
    if (warp == PRODUCER_WARP) {
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full, tiles * TILE_BYTES);
        for (int t = 0; t < tiles; ++t) issue_tile({smem + F_OFF_Q + t * TILE_BYTES, &map_q, q0 + t * 128, h, b}, q_full);
      }
      __syncwarp();
      const int rem = k_len < p.Sk ? k_len % 128 : 0;
      for (int seq = 0; seq < 2 * n; ++seq) {
        const int j = j0 + (seq >> 1);
        const uint32_t s = seq % F_SLOTS, ph = (seq / F_SLOTS) & 1u;
        if (!mbar_wait(&kv_empty[s], ph ^ 1u, abort_flag)) break;
        const TileLoad t = {smem + F_OFF_RING + s * TILE_BYTES, (seq & 1) ? &map_v : &map_k, j * 128, h, b};
        if (rem != 0 && j == n_all - 1 && (seq & 1) == 1) {
          if (!load_tile_tail(t, tail, 0, rem, &kv_full[s], abort_flag)) break;
        } else if (lane == 0) {
          mbar_arrive_expect_tx(&kv_full[s], TILE_BYTES);
          issue_tile(t, &kv_full[s]);
        }
        __syncwarp();
      }
    } else if (warp == ISSUER_WARP0) {
      const bool leader = elect_one();
      const uint32_t q_base = smem_u32(smem + F_OFF_Q), ring = smem_u32(smem + F_OFF_RING), id = idesc_k<BF16>();
      bool ok = mbar_wait(q_full, 0, abort_flag);
      for (int u = 0; ok && u < tiles * n; ++u) {  // use number u of the shared score buffer
        const int j = tiles == 2 ? u >> 1 : u, t = tiles == 2 ? u & 1 : 0;
        const uint32_t seq = 2 * j, s = seq % F_SLOTS, ph = (seq / F_SLOTS) & 1u;
        ok = mbar_wait(&kv_full[s], ph, abort_flag) && (u == 0 || mbar_wait(s_free, (u - 1) & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          mma_ss(tm, q_base + t * TILE_BYTES, ring + s * TILE_BYTES, id);
          umma_commit(&s_full[t]);
          umma_commit(&kv_empty[s]);
        }
        __syncwarp();
      }
    } else if (warp == ISSUER_WARP1) {
      const bool leader = elect_one();
      const uint32_t ring = smem_u32(smem + F_OFF_RING), id_mn = idesc_mn<BF16>();
      bool ok = true;
      for (int u = 0; ok && u < tiles * n; ++u) {
        const int j = tiles == 2 ? u >> 1 : u, t = tiles == 2 ? u & 1 : 0;
        const uint32_t seq = 2 * j + 1, s = seq % F_SLOTS, ph = (seq / F_SLOTS) & 1u;
        ok = mbar_wait(&kv_full[s], ph, abort_flag) && mbar_wait(&p_full[t], j & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          mma_ts_mn(tm + 256 + t * 128, tm + 128 + t * 64, 32, ring + s * TILE_BYTES, id_mn, j == 0);
          umma_commit(&pv_done[t]);
          umma_commit(&kv_empty[s]);
        }
        __syncwarp();
      }
    }
  } else if (x < tiles) {
    reg_alloc_216();
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tm + lanes, p_tmem = tm + lanes + 128 + x * 64, o_tmem = tm + lanes + 256 + x * 128;
    const float cmul = p.sm_scale * LOG2E;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      if (!(ok = mbar_wait(&s_full[x], j & 1u, abort_flag))) break;
      tc_fence_after_sync();
      uint32_t sv[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(s_tmem + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&sv[32 * c]));
      tmem_wait_ld();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free);
      const int valid = k_len - (j0 + j) * 128;
      if (valid < 128) {
#pragma unroll
        for (int i = 0; i < 128; ++i) sv[i] = i < valid ? sv[i] : 0xFF800000u;  // -inf: never the maximum, exp = 0
      }
      float fmx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 128; i += 2)
        fmx[(i >> 1) & 3] = fmax3(fmx[(i >> 1) & 3], __uint_as_float(sv[i]), __uint_as_float(sv[i + 1]));
      const float mx = fmaxf(fmax3(fmx[0], fmx[1], fmx[2]), fmx[3]) * cmul;  // cmul > 0
      const float m_new = (mx > m + TAU) ? mx : m;
      const float alpha = ex2(m - m_new);  // m = -inf on the first tile -> 0
      const float off = -m_new;
      if (j > 0) {
        if (!(ok = mbar_wait(&pv_done[x], (j - 1) & 1u, abort_flag))) break;
        tc_fence_after_sync();
      }
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t ov[32];
          tmem_ld32(o_tmem + 32 * c, ov);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
          tmem_st32(o_tmem + 32 * c, ov);
        }
      }
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int hseg = 0; hseg < 2; ++hseg) {
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const int i = 64 * hseg + 2 * c;
          const float e0 = ex2(fmaf(__uint_as_float(sv[i]), cmul, off));
          const float e1 = ex2(fmaf(__uint_as_float(sv[i + 1]), cmul, off));
          sum[c & 3] += e0;
          sum[(c + 2) & 3] += e1;
          pk[c] = pack_rn<BF16>(e0, e1);
        }
        tmem_st32(p_tmem + 32 * hseg, pk);
      }
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[x]);
      l = fmaf(l, alpha, (sum[0] + sum[1]) + (sum[2] + sum[3]));
      m = m_new;
    }
    if (ok && mbar_wait(&pv_done[x], (n - 1) & 1u, abort_flag)) {
      tc_fence_after_sync();
      const bool live = q_row < q_len;
      const float inv_l = 1.f / l, l2 = m + log2f(l);
      if (live) {
        if (p.splits > 1) p.part_lse[split_row] = l2;
        else p.lse[row] = l2 * LN2;
      }
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t ov[32];
        tmem_ld32(o_tmem + c * 32, ov);
        tmem_wait_ld();
        if (!live) continue;
        if (p.splits > 1) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(p.part + split_row * 128 + 32 * c + i) =
                make_float4(__uint_as_float(ov[i]) * inv_l, __uint_as_float(ov[i + 1]) * inv_l, __uint_as_float(ov[i + 2]) * inv_l,
                            __uint_as_float(ov[i + 3]) * inv_l);
        } else {
          store_row32<BF16>(out_ptr(p.o, b, h, q_row) + c * 32, ov, inv_l);
        }
      }
      if (!live) store_nothing();
    }
  } else {
    reg_dealloc_72();
    store_nothing();
  }
  close_tmem(tm, warp, abort_flag, p.status);
}

// ---- joins of split runs -------------------------------------------------------------------------------------------------
// One thread = four channels of a row; the parts are added in the order of the splits.
template <bool BF16>
__device__ __forceinline__ void store4(uint16_t* dst, float4 v, float mul) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_rn<BF16>(v.x * mul, v.y * mul), pack_rn<BF16>(v.z * mul, v.w * mul));
}
template <bool BF16>
__global__ void __launch_bounds__(256) attn_fwd_join_kernel(const TrainParams p) {
  const int64_t rows = static_cast<int64_t>(p.B) * p.heads * p.Sq;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32;
  if (row >= rows) return;
  const int c = (threadIdx.x & 31) * 4, bh = static_cast<int>(row / p.Sq), s = static_cast<int>(row % p.Sq);
  float top = -INFINITY;
  for (int k = 0; k < p.splits; ++k) {
    const float v = p.part_lse[k * rows + row];
    top = v > top || v != v ? v : top;  // a NaN stays
  }
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float total = 0.f;
  if (top != -INFINITY) {
    for (int k = 0; k < p.splits; ++k) {
      const float w = exp2f(p.part_lse[k * rows + row] - top);
      const float4 v = *reinterpret_cast<const float4*>(p.part + (k * rows + row) * 128 + c);
      total += w;
      acc.x = fmaf(w, v.x, acc.x);
      acc.y = fmaf(w, v.y, acc.y);
      acc.z = fmaf(w, v.z, acc.z);
      acc.w = fmaf(w, v.w, acc.w);
    }
  }
  store4<BF16>(out_ptr(p.o, bh / p.heads, bh % p.heads, s) + c, acc, top == -INFINITY ? 0.f : 1.f / total);
  if (c == 0) p.lse[row] = top == -INFINITY ? -INFINITY : (top + log2f(total)) * LN2;
}

struct JoinTarget { Rows out; const float* part; const int* k_lens; float mul; };
template <bool BF16>
__global__ void __launch_bounds__(256) attn_bwd_join_kernel(const JoinTarget t0, const JoinTarget t1, int splits, int64_t rows,
                                                            int S, int heads, int Sk) {
  const JoinTarget& t = blockIdx.y == 0 ? t0 : t1;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32;
  if (row >= rows) return;
  const int c = (threadIdx.x & 31) * 4, bh = static_cast<int>(row / S), s = static_cast<int>(row % S), b = bh / heads;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < splits; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(t.part + (k * rows + row) * 128 + c);
    acc.x += v.x;
    acc.y += v.y;
    acc.z += v.z;
    acc.w += v.w;
  }
  // t.mul 1: dv.  Otherwise a gradient through the scores, zero where there is one key only
  const float mul = t.k_lens == nullptr && Sk == 1 ? 0.f : t.k_lens != nullptr && valid_len(t.k_lens, b, Sk) == 1 ? 0.f : t.mul;
  store4<BF16>(out_ptr(t.out, b, bh % heads, s) + c, acc, mul);
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// Splits of the long axis.  `units` CTAs walk over `inner` tiles each; they run in waves of one CTA per SM, so a launch takes
// waves x (tiles per CTA + `fixed`), `fixed` being the prologue and epilogue of a CTA in tiles.  Splitting fills the last
// wave and, with few rows, the GPU, but its fp32 parts are written and read again: `join` tiles' time for each split of a
// whole wave's outputs.
inline int choose_splits(int64_t units, int64_t inner, double fixed, double join) {
  const int64_t sms = sm_count();
  int best = 1;
  double best_cost = 0;
  for (int s = 1; s <= kMaxSplits && (s == 1 || inner >= 2 * s); ++s) {
    const double waves = static_cast<double>((units * s + sms - 1) / sms);
    const double cost = waves * (static_cast<double>((inner + s - 1) / s) + fixed) + (s > 1 ? 4.0 + join * static_cast<double>(units * s) / sms : 0.0);
    if (s == 1 || cost < 0.97 * best_cost) {
      best = s;
      best_cost = cost;
    }
  }
  return best;
}
inline int64_t tiles_of(int64_t S, int64_t t) { return (S + t - 1) / t; }
inline int forward_splits(int64_t BH, int64_t Sq, int64_t Sk) { return choose_splits(BH * tiles_of(Sq, 256), tiles_of(Sk, 128), 3.0, 0.6); }
inline int dq_splits(int64_t BH, int64_t Sq, int64_t Sk) { return choose_splits(BH * tiles_of(Sq, 128), tiles_of(Sk, 128), 4.0, 0.3); }
inline int dkdv_splits(int64_t BH, int64_t Sq, int64_t Sk) { return choose_splits(BH * tiles_of(Sk, 128), tiles_of(Sq, 128), 4.0, 0.6); }
inline int64_t pad128(int64_t S) { return tiles_of(S, 128) * 128; }
inline size_t round256(size_t n) { return (n + 255) / 256 * 256; }

struct BackwardLayout { size_t stats, dq, dkdv, bytes; };
inline BackwardLayout backward_layout(int64_t BH, int64_t Sq, int64_t Sk) {
  BackwardLayout w{};
  const int s_q = dq_splits(BH, Sq, Sk), s_kv = dkdv_splits(BH, Sq, Sk);
  w.stats = 0;
  w.dq = round256(static_cast<size_t>(BH) * pad128(Sq) * 8);
  w.dkdv = w.dq + (s_q > 1 ? round256(static_cast<size_t>(s_q) * BH * Sq * 512) : 0);
  w.bytes = w.dkdv + (s_kv > 1 ? round256(static_cast<size_t>(s_kv) * BH * Sk * 1024) : 0);
  return w;
}

int check_shape(const char* what, int dtype, int64_t B, int64_t heads, int64_t Sq, int64_t Sk, float sm_scale) {
  DAX_REQUIRE(B > 0 && heads > 0 && Sq > 0 && Sk > 0, DAX_ERR_INVALID, "%s: bad shape B=%lld heads=%lld Sq=%lld Sk=%lld", what,
              (long long)B, (long long)heads, (long long)Sq, (long long)Sk);
  DAX_REQUIRE(dtype == DAX_BF16 || dtype == DAX_F16, DAX_ERR_UNSUPPORTED, "%s: dtype %d is not BF16/F16", what, dtype);
  DAX_REQUIRE(B * heads <= 65535, DAX_ERR_UNSUPPORTED, "%s: batch*heads=%lld exceeds 65535", what, (long long)(B * heads));
  DAX_REQUIRE(Sq < (1ll << 30) && Sk < (1ll << 30), DAX_ERR_UNSUPPORTED, "%s: sequence too long", what);
  DAX_REQUIRE(std::isfinite(sm_scale) && sm_scale > 0.f, DAX_ERR_INVALID, "%s: the softmax scale must be positive and finite", what);
  return DAX_OK;
}
int check_rows(const char* what, const char* name, const void* t, const int64_t* st) {
  DAX_REQUIRE(t != nullptr && st != nullptr, DAX_ERR_INVALID, "%s: %s is null", what, name);
  DAX_REQUIRE(aligned16(t) && st[0] % 8 == 0 && st[1] % 8 == 0 && st[2] % 8 == 0, DAX_ERR_ALIGN,
              "%s: %s must be 16-byte aligned with strides that are multiples of 8 elements", what, name);
  DAX_REQUIRE(st[0] >= 0 && st[1] >= 0 && st[2] >= 0, DAX_ERR_INVALID, "%s: %s has a negative stride", what, name);
  return DAX_OK;
}
// [128 channels, S, heads, B] map with boxes of [64 channels x 128 tokens]
int make_map(CUtensorMap* m, const void* t, const int64_t* st, int64_t S, int64_t heads, int64_t B) {
  const uint64_t dims[4] = {128, static_cast<uint64_t>(S), static_cast<uint64_t>(heads), static_cast<uint64_t>(B)};
  uint64_t strides[4] = {2, static_cast<uint64_t>(st[2]) * 2, static_cast<uint64_t>(st[1]) * 2, static_cast<uint64_t>(st[0]) * 2};
  for (int i = 1; i < 4; ++i) {
    if (dims[i] == 1) strides[i] = 256;  // never used, but the encoder wants a valid one
    DAX_REQUIRE(strides[i] > 0 && strides[i] < (1ull << 40), DAX_ERR_INVALID, "attention: a stride of %llu bytes cannot be addressed",
                (unsigned long long)strides[i]);
  }
  const uint32_t box[4] = {64, 128, 1, 1};
  return make_tma_map(m, t, 2, 4, dims, strides, box);
}
inline Rows rows_of(const void* t, const int64_t* st) { return {t, st[0], st[1], st[2]}; }

#define DAX_TRY(expr)              \
  do {                             \
    const int rc__ = (expr);       \
    if (rc__ != DAX_OK) return rc__; \
  } while (0)

template <bool BF16>
int run_forward(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const TrainParams& p, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(tiles_of(p.Sq, 256)), static_cast<unsigned>(p.B * p.heads), static_cast<unsigned>(p.splits));
  DAX_CUDA(cudaFuncSetAttribute(attn_fwd_lse_kernel<BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, F_SMEM));
  attn_fwd_lse_kernel<BF16><<<grid, THREADS, F_SMEM, st>>>(mq, mk, mv, p);
  DAX_CUDA(cudaGetLastError());
  if (p.splits > 1) {
    attn_fwd_join_kernel<BF16><<<static_cast<unsigned>(tiles_of(static_cast<int64_t>(p.B) * p.heads * p.Sq, 8)), 256, 0, st>>>(p);
    DAX_CUDA(cudaGetLastError());
  }
  return DAX_OK;
}

template <bool BF16>
int run_backward(const CUtensorMap& mq, const CUtensorMap& mdo, const CUtensorMap& mk, const CUtensorMap& mv, TrainParams p,
                 int s_q, int s_kv, float* part_q, float* part_kv, cudaStream_t st) {
  const unsigned BH = static_cast<unsigned>(p.B * p.heads);
  p.splits = s_q;
  p.part = part_q;
  DAX_CUDA(cudaFuncSetAttribute(attn_bwd_dq_kernel<BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, DQ_SMEM));
  attn_bwd_dq_kernel<BF16><<<dim3(static_cast<unsigned>(tiles_of(p.Sq, 128)), BH, static_cast<unsigned>(s_q)), THREADS, DQ_SMEM, st>>>(mk, mv, p);
  DAX_CUDA(cudaGetLastError());
  if (s_q > 1) {
    const int64_t rows = static_cast<int64_t>(BH) * p.Sq;
    const JoinTarget t = {p.dq, part_q, p.k_lens, p.sm_scale};
    attn_bwd_join_kernel<BF16><<<dim3(static_cast<unsigned>(tiles_of(rows, 8)), 1), 256, 0, st>>>(t, t, s_q, rows, p.Sq, p.heads, p.Sk);
    DAX_CUDA(cudaGetLastError());
  }
  p.splits = s_kv;
  p.part = part_kv;
  DAX_CUDA(cudaFuncSetAttribute(attn_bwd_dkdv_kernel<BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, KV_SMEM));
  attn_bwd_dkdv_kernel<BF16><<<dim3(static_cast<unsigned>(tiles_of(p.Sk, 128)), BH, static_cast<unsigned>(s_kv)), THREADS, KV_SMEM, st>>>(mq, mdo, mk, mv, p);
  DAX_CUDA(cudaGetLastError());
  if (s_kv > 1) {
    const int64_t rows = static_cast<int64_t>(BH) * p.Sk;
    const JoinTarget tk = {p.dk, part_kv, p.k_lens, p.sm_scale}, tv = {p.dv, part_kv + s_kv * rows * 128, nullptr, 1.f};
    attn_bwd_join_kernel<BF16><<<dim3(static_cast<unsigned>(tiles_of(rows, 8)), 2), 256, 0, st>>>(tk, tv, s_kv, rows, p.Sk, p.heads, p.Sk);
    DAX_CUDA(cudaGetLastError());
  }
  return DAX_OK;
}

}  // namespace
}  // namespace dax

extern "C" {

size_t dax_attn_lse_workspace_bytes(int64_t B, int64_t heads, int64_t Sq, int64_t Sk) {
  using namespace dax;
  if (B <= 0 || heads <= 0 || Sq <= 0 || Sk <= 0) return 0;
  const int s = forward_splits(B * heads, Sq, Sk);
  return s > 1 ? static_cast<size_t>(s) * B * heads * Sq * (512 + 4) : 0;
}

int dax_attn_forward_lse(const void* q, const void* k, const void* v, int dtype, int64_t B, int64_t heads, int64_t Sq, int64_t Sk,
                         int64_t q_strides[3], int64_t k_strides[3], int64_t v_strides[3], float sm_scale, const int32_t* q_lens,
                         const int32_t* k_lens, void* o, int64_t o_strides[3], float* lse, void* workspace, size_t workspace_bytes,
                         void* stream) {
  using namespace dax;
  const char* what = "attn_forward_lse";
  DAX_TRY(check_shape(what, dtype, B, heads, Sq, Sk, sm_scale));
  DAX_TRY(check_rows(what, "q", q, q_strides));
  DAX_TRY(check_rows(what, "k", k, k_strides));
  DAX_TRY(check_rows(what, "v", v, v_strides));
  DAX_TRY(check_rows(what, "o", o, o_strides));
  DAX_REQUIRE(lse != nullptr, DAX_ERR_INVALID, "%s: lse is null", what);
  const size_t need = dax_attn_lse_workspace_bytes(B, heads, Sq, Sk);
  DAX_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), DAX_ERR_INVALID,
              "%s: workspace of %zu bytes is smaller than the %zu required", what, workspace_bytes, need);
  DAX_REQUIRE(need == 0 || aligned16(workspace), DAX_ERR_ALIGN, "%s: workspace must be 16-byte aligned", what);
  CUtensorMap mq, mk, mv;
  DAX_TRY(make_map(&mq, q, q_strides, Sq, heads, B));
  DAX_TRY(make_map(&mk, k, k_strides, Sk, heads, B));
  DAX_TRY(make_map(&mv, v, v_strides, Sk, heads, B));
  TrainParams p{};
  p.o = rows_of(o, o_strides);
  p.lse = lse;
  p.q_lens = q_lens;
  p.k_lens = k_lens;
  p.splits = forward_splits(B * heads, Sq, Sk);
  p.part = static_cast<float*>(workspace);
  p.part_lse = p.part + static_cast<int64_t>(p.splits) * B * heads * Sq * 128;
  p.status = device_status_ptr();
  DAX_REQUIRE(p.status != nullptr, DAX_ERR_CUDA, "%s: cannot resolve the device status word", what);
  p.B = static_cast<int>(B);
  p.heads = static_cast<int>(heads);
  p.Sq = static_cast<int>(Sq);
  p.Sk = static_cast<int>(Sk);
  p.sm_scale = sm_scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == DAX_BF16 ? run_forward<true>(mq, mk, mv, p, st) : run_forward<false>(mq, mk, mv, p, st);
}

size_t dax_attn_backward_workspace_bytes(int64_t B, int64_t heads, int64_t Sq, int64_t Sk) {
  if (B <= 0 || heads <= 0 || Sq <= 0 || Sk <= 0) return 0;
  return dax::backward_layout(B * heads, Sq, Sk).bytes;
}

int dax_attn_backward(const void* dout, const void* q, const void* k, const void* v, const void* o, const float* lse, int dtype,
                      int64_t B, int64_t heads, int64_t Sq, int64_t Sk, int64_t do_strides[3], int64_t q_strides[3],
                      int64_t k_strides[3], int64_t v_strides[3], int64_t o_strides[3], float sm_scale, const int32_t* q_lens,
                      const int32_t* k_lens, void* dq, void* dk, void* dv, int64_t dq_strides[3], int64_t dk_strides[3],
                      int64_t dv_strides[3], void* workspace, size_t workspace_bytes, void* stream) {
  using namespace dax;
  const char* what = "attn_backward";
  DAX_TRY(check_shape(what, dtype, B, heads, Sq, Sk, sm_scale));
  DAX_TRY(check_rows(what, "dout", dout, do_strides));
  DAX_TRY(check_rows(what, "q", q, q_strides));
  DAX_TRY(check_rows(what, "k", k, k_strides));
  DAX_TRY(check_rows(what, "v", v, v_strides));
  DAX_TRY(check_rows(what, "o", o, o_strides));
  DAX_TRY(check_rows(what, "dq", dq, dq_strides));
  DAX_TRY(check_rows(what, "dk", dk, dk_strides));
  DAX_TRY(check_rows(what, "dv", dv, dv_strides));
  DAX_REQUIRE(lse != nullptr, DAX_ERR_INVALID, "%s: lse is null", what);
  const BackwardLayout w = backward_layout(B * heads, Sq, Sk);
  DAX_REQUIRE(workspace != nullptr && workspace_bytes >= w.bytes, DAX_ERR_INVALID,
              "%s: workspace of %zu bytes is smaller than the %zu required", what, workspace_bytes, w.bytes);
  DAX_REQUIRE(aligned16(workspace), DAX_ERR_ALIGN, "%s: workspace must be 16-byte aligned", what);
  CUtensorMap mq, mdo, mk, mv;
  DAX_TRY(make_map(&mq, q, q_strides, Sq, heads, B));
  DAX_TRY(make_map(&mdo, dout, do_strides, Sq, heads, B));
  DAX_TRY(make_map(&mk, k, k_strides, Sk, heads, B));
  DAX_TRY(make_map(&mv, v, v_strides, Sk, heads, B));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  TrainParams p{};
  p.q = rows_of(q, q_strides);
  p.o = rows_of(o, o_strides);
  p.dout = rows_of(dout, do_strides);
  p.dq = rows_of(dq, dq_strides);
  p.dk = rows_of(dk, dk_strides);
  p.dv = rows_of(dv, dv_strides);
  p.lse = const_cast<float*>(lse);
  p.q_lens = q_lens;
  p.k_lens = k_lens;
  p.row_stats = reinterpret_cast<float*>(ws + w.stats);
  p.status = device_status_ptr();
  DAX_REQUIRE(p.status != nullptr, DAX_ERR_CUDA, "%s: cannot resolve the device status word", what);
  p.B = static_cast<int>(B);
  p.heads = static_cast<int>(heads);
  p.Sq = static_cast<int>(Sq);
  p.Sk = static_cast<int>(Sk);
  p.Sq_pad = static_cast<int>(pad128(Sq));
  p.sm_scale = sm_scale;
  const int s_q = dq_splits(B * heads, Sq, Sk), s_kv = dkdv_splits(B * heads, Sq, Sk);
  float* part_q = reinterpret_cast<float*>(ws + w.dq);
  float* part_kv = reinterpret_cast<float*>(ws + w.dkdv);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == DAX_BF16 ? run_backward<true>(mq, mdo, mk, mv, p, s_q, s_kv, part_q, part_kv, st)
                           : run_backward<false>(mq, mdo, mk, mv, p, s_q, s_kv, part_q, part_kv, st);
}

}  // extern "C"
