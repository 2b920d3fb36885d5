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
// Bound by the tensor cores and, in long runs, by power (the SM clock falls to 1.65 GHz).  Measured, bf16: forward 1,215
// TFLOP/s at 5 heads x 16,384 tokens (566 us), 1,240 at 40 x 4,096; backward 943 and 900 TFLOP/s of its own ten operations per
// pair and channel, 1,320 and 1,260 of the fourteen that the seven products do (1,821 and 955 us; fp16 1,945 and 1,035).  A library product
// of 16-bit matrices reaches 1,615 for a moment and 1,373 for seconds.
//
// q_lens / k_lens (per sample, optional) bound the tokens that exist: rows behind a length take no part in anything (not
// even when they hold NaN or infinity), their outputs are zero and their lse is -inf, and so are those of queries that
// see no key at all.
//
// Scores, probabilities, row statistics, D and all sums are fp32.  p and ds are rounded once to the operands' type, as A
// operands of the second products (the tensor cores take nothing wider together with 16-bit B operands).  fp16 has its
// smallest normal number at 2^-14, and the p of a long row of keys, or of keys beside a dominant one, lie below it: the
// backward pass rounds 2^12 p, which is normal down to p = 2^-26, and takes the factor out of dv again; the forward pass rounds
// 2^11 p / max p (F_SHIFT), and its factor leaves with the row's sum.  ds is smaller than do by a factor of p as well, and larger by
// that of v; |ds_ij| <= 2 |do_i| max_j |v_j| bounds it.  In fp16 it is rounded times the power of two that brings this bound to
// 2^15: one for each query in dq (it leaves with the row), one for each head in dk, whose sums run over the queries.  Error of dq
// of 32,760 keys (in brackets one rounding of the exact result), ds rounded as it is / with the factors: do of 1e-2 3.0e-3 /
// 3.0e-4 (2.1e-4), 1e-3 3.0e-2 / 5.2e-4 (4.7e-4: results below 2^-14); infinite / finite where ds passes 65,504.  A small kernel
// finds the largest norms first (fp16 only).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "quant_common.cuh"
#include "sm100_ptx.cuh"

namespace dax {
namespace {

constexpr int BOX_BYTES = 128 * 128;       // one [128 rows x 64 channels] box
constexpr int TILE_BYTES = 2 * BOX_BYTES;  // a [128 x 128] tile of 16-bit elements
// Warps: N row warps (all arithmetic on scores), then a TMA producer, two issuers of products, the owner of tensor memory.
constexpr int ROW_WARPS_F = 8, ROW_WARPS_B = 16;
template <int N> struct Warps {
  static constexpr int threads = (N + 4) * 32, producer = N, issuer0 = N + 1, issuer1 = N + 2, tmem = N + 3;
};
// Forward: the sums are rescaled when the row's maximum has risen by more than 2^TAU, so p (relative to the maximum then) is at
// most 2^TAU; it is rounded as 2^F_SHIFT p, and so is its sum taken.  fp16: at most 2^15, and normal down to 2^-25 of the largest.
template <bool BF16> constexpr float TAU = BF16 ? 8.f : 4.f;
template <bool BF16> constexpr float F_SHIFT = BF16 ? 0.f : 11.f;
template <bool BF16> constexpr float P_SHIFT = BF16 ? 0.f : 12.f;             // backward: p is rounded as 2^P_SHIFT p
template <bool BF16> constexpr float P_UNSHIFT = BF16 ? 1.f : 1.f / 4096.f;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int kMaxSplits = 16;
constexpr int kRangeChunks = 32;  // of a head's tokens, for the largest norms: one per lane

struct Rows { const void* p; int64_t sb, sh, st; };  // a [B, heads, S, 128] view: element strides of sample, head, token

struct TrainParams {
  Rows o, dq, dk, dv;
  float* lse;          // [BH, Sq]
  const int* q_lens;   // [B] or null
  const int* k_lens;
  float* row_stats;    // backward: [2][BH * Sq_pad]: P_SHIFT - lse * log2(e) (-inf: no such row), then -D * P_UNSHIFT
  float* range;        // backward, fp16: [2][BH][kRangeChunks]: largest |v_j|^2, then largest |do_i|^2, of each chunk of the head's tokens
  float* part;         // split runs: fp32 partial sums
  float* part_lse;     // split forward runs: [splits, BH, Sq] log2 of each part's sum of exponentials
  float* part_e;       // split dq runs: [splits, BH, Sq_pad] sums of ds, as row_stats has D
  int* status;
  int B, heads, Sq, Sk, Sq_pad, splits;
  float sm_scale;
};

// Register split: row warps and the others, together what the block was launched with (12 warps x 168, 20 warps x 96)
template <int N> __device__ __forceinline__ void row_warp_registers() {
  if constexpr (N == ROW_WARPS_F) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
}
template <int N> __device__ __forceinline__ void other_warp_registers() {
  if constexpr (N == ROW_WARPS_F) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
}

// acc += both halves of a pair of rounded values
template <bool BF16>
__device__ __forceinline__ void add_pair(float& acc, uint32_t w) {
  if constexpr (BF16)
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tadd.rn.f32.bf16 %0, l, %0;\n\tadd.rn.f32.bf16 %0, h, %0;\n\t}" : "+f"(acc) : "r"(w));
  else
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tadd.rn.f32.f16 %0, l, %0;\n\tadd.rn.f32.f16 %0, h, %0;\n\t}" : "+f"(acc) : "r"(w));
}
__device__ __forceinline__ uint64_t f2_bits(uint32_t lo, uint32_t hi) { return f2_pack(__uint_as_float(lo), __uint_as_float(hi)); }
__device__ __forceinline__ int valid_len(const int* lens, int b, int S) { return lens != nullptr ? min(max(lens[b], 0), S) : S; }

__device__ __forceinline__ const uint16_t* row_ptr(const Rows& t, int b, int h, int64_t s) {
  return static_cast<const uint16_t*>(t.p) + b * t.sb + h * t.sh + s * t.st;
}
__device__ __forceinline__ uint16_t* out_ptr(const Rows& t, int b, int h, int64_t s) { return const_cast<uint16_t*>(row_ptr(t, b, h, s)); }

// ---- results to memory ----------------------------------------------------------------------------------------------
// A thread holds a row, memory wants whole lines: a warp's 32 rows x ROWB bytes (64 or 128) go through its own piece of shared
// memory, 16-byte chunks permuted so that neither side has bank conflicts.
template <int ROWB>
__device__ __forceinline__ uint4* stage_at(uint8_t* st, int row, int chunk) {
  const int swz = ROWB == 128 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3);
  return reinterpret_cast<uint4*>(st + row * ROWB + swz * 16);
}
template <int ROWB>
__device__ __forceinline__ void stage_flush(uint8_t* st, uint8_t* dst, int64_t row_bytes, int rows) {
  constexpr int L = ROWB / 16;
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int row = (i * 32 + lane) / L, chunk = lane % L;
    if (row < rows) *reinterpret_cast<uint4*>(dst + row * row_bytes + chunk * 16) = *stage_at<ROWB>(st, row, chunk);
  }
  __syncwarp();
}
// 32 columns of the warp's rows, times `mul`, rounded (64 bytes per row) ...
template <bool BF16>
__device__ __forceinline__ void store_cols32(uint8_t* st, const uint32_t (&v)[32], float mul, bool live, uint16_t* dst, int64_t row_elements, int rows) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = pack2_rn<BF16>(__uint_as_float(v[8 * c + 2 * k]) * mul, __uint_as_float(v[8 * c + 2 * k + 1]) * mul);
    *stage_at<64>(st, threadIdx.x & 31, c) = live ? make_uint4(w[0], w[1], w[2], w[3]) : make_uint4(0u, 0u, 0u, 0u);
  }
  stage_flush<64>(st, reinterpret_cast<uint8_t*>(dst), row_elements * 2, rows);
}
// ... or as fp32 parts of a split run (128 bytes per row, rows of 128 floats)
__device__ __forceinline__ void store_part32(uint8_t* st, const uint32_t (&v)[32], float mul, bool live, float* dst, int rows) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = live ? __float_as_uint(__uint_as_float(v[4 * c + k]) * mul) : 0u;
    *stage_at<128>(st, threadIdx.x & 31, c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  stage_flush<128>(st, reinterpret_cast<uint8_t*>(dst), 512, rows);
}
// `rows` rows of `bytes` zeros, by the whole block
__device__ __forceinline__ void zero_rows(void* dst, int64_t row_bytes, int rows, int bytes) {
  const int chunks = bytes / 16;
  for (int i = threadIdx.x; i < rows * chunks; i += blockDim.x)
    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(dst) + (i / chunks) * row_bytes + (i % chunks) * 16) = make_uint4(0u, 0u, 0u, 0u);
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
// D += A[tmem] . B[smem] with the contraction over the tile's rows: B is MN-major, 16 rows per step
__device__ __forceinline__ void mma_ts_mn(uint32_t d, uint32_t a_tmem, uint32_t b_smem, uint32_t idesc, bool first) {
  const uint64_t b = make_desc_mn_sw128(b_smem, BOX_BYTES);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    umma_ts_f16(d, a_tmem + 8 * i, b + static_cast<uint64_t>(i * ((16 * 128) >> 4)), idesc,
                (!first || i != 0) ? 1u : 0u);
}
template <bool BF16>
__device__ __forceinline__ uint32_t idesc_k() { return make_idesc(1, BF16 ? 1 : 0, BF16 ? 1 : 0, 128, 128); }
template <bool BF16>
__device__ __forceinline__ uint32_t idesc_mn() { return idesc_k<BF16>() | (1u << 16); }  // B is MN-major

// Half `c` of such a product whose A operand comes from four row warps, each with 16 columns for 32 of the tile's rows: the
// first (c = 0) or the second 16 rows of each.
__device__ __forceinline__ void mma_ts_mn_half(uint32_t d, uint32_t a_tmem, int c, uint32_t b_smem, uint32_t idesc, bool first) {
  const uint64_t b = make_desc_mn_sw128(b_smem, BOX_BYTES);
#pragma unroll
  for (int g = 0; g < 4; ++g)
    umma_ts_f16(d, a_tmem + 16 * g + 8 * c, b + static_cast<uint64_t>((2 * g + c) * ((16 * 128) >> 4)), idesc, (!first || g != 0) ? 1u : 0u);
}

// Set-up and tear-down shared by the kernels
__device__ __forceinline__ uint32_t open_tmem(uint32_t* slot, bool owner) {
  if (owner) {
    tmem_alloc(slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  return *slot;
}
__device__ __forceinline__ void close_tmem(uint32_t base, bool owner, volatile uint32_t* abort_flag, int* status) {
  if (*abort_flag)  // a wait gave up: copies and products in flight land (a millisecond) before the block returns its memory
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  tc_fence_before_sync();
  __syncthreads();
  if (owner) {
    tc_fence_after_sync();
    tmem_dealloc(base, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) atomicExch(status, DAX_ERR_TIMEOUT);
}

// ---- factors of ds in fp16 ---------------------------------------------------------------------------------------------
__host__ __device__ __forceinline__ int range_rows(int S) { return ((S + kRangeChunks - 1) / kRangeChunks + 15) / 16 * 16; }  // of a chunk
// The power of two that brings 2 |do| |v| to [2^14, 2^15), from the product of the squares; finite for 0 and infinity too.
__device__ __forceinline__ float range_factor(float squares) {
  const int e = static_cast<int>(__float_as_uint(4.f * squares) >> 23) - 127;  // 4 squares < 2^(e + 1)
  return __uint_as_float(static_cast<uint32_t>(127 + 15 - ((e + 2) >> 1)) << 23);
}
__device__ __forceinline__ float power_inverse(float f) { return __uint_as_float((254u << 23) - __float_as_uint(f)); }
// The largest of a head's squares over its chunks, by the whole warp (none is negative, so their bits order like numbers).
__device__ __forceinline__ float range_max(const float* range, int S) {
  const int lane = threadIdx.x & 31;
  const float v = lane * range_rows(S) < S ? range[lane] : 0.f;
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}
__device__ __forceinline__ float range_of_v(const TrainParams& p, int bh) { return range_max(p.range + static_cast<int64_t>(bh) * kRangeChunks, p.Sk); }
// A head's factor in dk, over that of p beside it: what -D is kept times for the dk/dv kernel.
__device__ __forceinline__ float stat_factor(const TrainParams& p, int bh) {
  const float do_top = range_max(p.range + (static_cast<int64_t>(p.B) * p.heads + bh) * kRangeChunks, p.Sq);
  return range_factor(do_top * range_of_v(p, bh)) * P_UNSHIFT<false>;
}

// Largest |v_j|^2 (blockIdx.z 0) and |do_i|^2 (1) of each chunk of tokens that exist: half a warp per token.  A NaN is passed
// over: what it touches is NaN anyway.  12 heads x 4,095 x 4,095: 10 us for 25 MB from DRAM (most of it latency; eight loads in
// flight instead of four change nothing), the backward pass takes 316 us with it and the factors, 307 without.
__global__ void __launch_bounds__(256) attn_range_kernel(const Rows v, const Rows dout, const TrainParams p) {
  const bool keys = blockIdx.z == 0;
  const Rows& t = keys ? v : dout;
  const int bh = blockIdx.y, b = bh / p.heads, h = bh % p.heads, S = keys ? p.Sk : p.Sq;
  const int per = range_rows(S), row0 = static_cast<int>(blockIdx.x) * per;
  if (row0 >= S) return;
  const int end = min(valid_len(keys ? p.k_lens : p.q_lens, b, S), row0 + per);
  const int piece = threadIdx.x & 15;
  float top = 0.f;
#pragma unroll 4
  for (int s = row0 + (threadIdx.x >> 4); s < row0 + per; s += 16) {  // the same number of steps for all threads
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (s < end) u = *reinterpret_cast<const uint4*>(row_ptr(t, b, h, s) + piece * 8);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    float n = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float a, c;
      unpack2<false>(w[k], a, c);
      n = fmaf(a, a, fmaf(c, c, n));
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    top = fmaxf(top, n);
  }
  __shared__ float tops[8];
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < 8; ++k) top = fmaxf(top, tops[k]);
    p.range[(static_cast<int64_t>(blockIdx.z) * p.B * p.heads + bh) * kRangeChunks + blockIdx.x] = top;
  }
}

// ---- dq ----------------------------------------------------------------------------------------------------------------
// One CTA = 128 query rows of one head, walking over the tiles of keys.
//   warps 0..15  one thread = one query row x 32 keys of the tile (warp / 4: which 32).  Two teams of eight take turns with
//                the exponentials (a token goes back and forth): one team's wait for the unit that computes them, the other's
//                for the multiply-add pipe and for tensor memory, fall into each other
//   producer     q, and do and o in the ring's last two slots; then k_0, v_0, k_1, ... through the ring, at last k's first tile
//   issuer 0     s = q.k_j^T and dp = do.v_j^T        issuer 1     dq += ds.k_j
// 8 heads x 4,096 x 4,096 bf16: 97 us, 1.3 us per tile of keys and CTA and about 6 us around them; tensor pipe 66 % of the
// time, unit of the exponentials 45 %.
// Tensor memory: s [0,128)  dp [128,256)  dq [256,384)  do [384,448)  ds [448,512).  do and ds are A operands in tensor
// memory, so of the three products only s reads both operands from shared memory, whose bandwidth would otherwise be the
// bound.  s and dp are free as soon as they are in registers, and ds has columns of its own: the next tile's products
// never wait for this tile's arithmetic.
//
// Keys often share an offset (the mean of trained keys is far from zero).  sum_j ds_ij is zero, so the offset has no part in
// dq, but the roundings of ds have: their sum times the offset would be the largest error by far.  The kernel adds up the
// rounded ds of each row, e_i, and subtracts e_i m for an m near the mean key (the first tile's), which is what rounding
// left of it.
//
// D is taken from the rounded o.  What that rounding leaves in ds is p_ij times one number per row, and that number is e_i (the
// exact ds of a row add up to zero): nothing beside the rounding of ds where a row spreads over many keys, more than it
// where p_ij is near one.  Where all keys lie in one tile the kernel has e_i before it rounds ds, and takes it out of D.  With
// more keys e_i is known at the end: the dk/dv kernel gets D + e_i, but dq keeps e_i times (the row's own mean of k - m), for
// which the sum of p_ij k_j would be needed, one product more.  Error of the norms of dq / dk, bf16, 1,000 x 2,000, in brackets one
// rounding of the exact result (1.7e-3): scores of unit spread 2.4e-3 / 2.3e-3, of spread 10 (largest p 0.74 on average) 5.2e-3 /
// 2.7e-3 (dk 5.0e-3 with D alone), of 30 (0.91) 6.4e-3 / 2.6e-3 (6.1e-3); fp16 an eighth of all.
constexpr int DQ_SLOTS = 6;
constexpr int DQ_OFF_Q = DQ_SLOTS * TILE_BYTES;
constexpr int DQ_OFF_MEAN = DQ_OFF_Q;               // [16][128] floats: sums of keys, in the end m in the first row; over q
constexpr int DQ_OFF_BAR = DQ_OFF_Q + TILE_BYTES;
constexpr int DQ_SMEM = DQ_OFF_BAR + 256 + 1024;
static_assert(DQ_SMEM <= 227 * 1024, "shared memory of the dq kernel");

__device__ __forceinline__ void row_warps_sync() { asm volatile("bar.sync 1, 512;" ::: "memory"); }  // warps 0..15

// The four column groups' values of a row, left in tensor memory 32 columns apart.
__device__ __forceinline__ float sum_of_groups(uint32_t taddr) {
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) tmem_ld1(taddr + 32 * i, v[i]);
  tmem_wait_ld();
  return (__uint_as_float(v[0]) + __uint_as_float(v[1])) + (__uint_as_float(v[2]) + __uint_as_float(v[3]));
}

template <bool BF16>
__global__ void __launch_bounds__(Warps<ROW_WARPS_B>::threads, 1)
attn_bwd_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                   const __grid_constant__ CUtensorMap map_o, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const TrainParams p) {
  using W = Warps<ROW_WARPS_B>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q0 = blockIdx.x * 128, bh = blockIdx.y, b = bh / p.heads, h = bh % p.heads, split = blockIdx.z;
  const int q_len = valid_len(p.q_lens, b, p.Sq), k_len = valid_len(p.k_lens, b, p.Sk);
  const int n_all = q0 < q_len ? (k_len + 127) / 128 : 0;
  const int per = (n_all + p.splits - 1) / p.splits;
  const int j0 = split * per, n = max(0, min(n_all, j0 + per) - j0);
  // a split run leaves fp32 sums [split][BH][Sq][128] that are joined afterwards
  float* part = p.part + ((static_cast<int64_t>(split) * p.B * p.heads + bh) * p.Sq + q0) * 128;
  float* stat = p.row_stats + static_cast<int64_t>(bh) * p.Sq_pad + q0;
  const auto part_e = [&] { return p.part_e + (static_cast<int64_t>(split) * p.B * p.heads + bh) * p.Sq_pad + q0; };
  const int64_t stats = static_cast<int64_t>(p.B) * p.heads * p.Sq_pad;
  const int rows_in = min(128, p.Sq - q0);  // rows of the CTA

  if (n == 0) {  // nothing to see: zeros
    if (split == 0 && threadIdx.x < 128) {
      stat[threadIdx.x] = -INFINITY;
      stat[stats + threadIdx.x] = 0.f;
    }
    if (p.splits > 1 && threadIdx.x < 128) part_e()[threadIdx.x] = 0.f;
    if (p.splits > 1) zero_rows(part, 512, rows_in, 512);
    else zero_rows(out_ptr(p.dq, b, h, q0), p.dq.st * 2, rows_in, 256);
    return;
  }

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + DQ_OFF_BAR);
  uint64_t* full = bars;                 // [DQ_SLOTS]
  uint64_t* empty = full + DQ_SLOTS;     // [DQ_SLOTS] k: released by dq; v: by dp
  uint64_t* tail = empty + DQ_SLOTS;
  uint64_t* q_full = tail + 1;           // q in shared memory
  uint64_t* rows_full = q_full + 1;      // do and o in shared memory
  uint64_t* do_full = rows_full + 1;     // do and the parts of D in tensor memory
  uint64_t* s_full = do_full + 1;
  uint64_t* s_free = s_full + 1;
  uint64_t* dp_full = s_free + 1;
  uint64_t* dp_free = dp_full + 1;
  uint64_t* ds_full = dp_free + 1;
  uint64_t* dq_done = ds_full + 1;
  uint64_t* turn = dq_done + 1;          // [2]
  uint64_t* sums_full = turn + 2;        // one tile of keys: the column groups' sums are in tensor memory
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sums_full + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  uint8_t* do_smem = smem + (DQ_SLOTS - 2) * TILE_BYTES;
  uint8_t* o_smem = smem + (DQ_SLOTS - 1) * TILE_BYTES;
  const int rem = k_len < p.Sk ? k_len % 128 : 0;  // tokens of the last tile that exist (0: no tail of k to clear)
  const bool early = !(rem != 0 && n_all == j0 + 1);  // the first tile of k has no tail to clear
  if (warp == W::producer && lane == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_do);
    tma_prefetch_desc(&map_o);
    tma_prefetch_desc(&map_v);
    for (int i = 0; i < DQ_SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(tail, 1);
    mbar_init(q_full, 1);
    mbar_init(rows_full, 1);
    mbar_init(do_full, ROW_WARPS_B);
    mbar_init(s_full, 1);
    mbar_init(s_free, ROW_WARPS_B);
    mbar_init(dp_full, 1);
    mbar_init(dp_free, ROW_WARPS_B);
    mbar_init(ds_full, ROW_WARPS_B);
    mbar_init(dq_done, 1);
    mbar_init(&turn[0], ROW_WARPS_B / 2);
    mbar_init(&turn[1], ROW_WARPS_B / 2);
    mbar_init(sums_full, ROW_WARPS_B);
    *abort_flag = 0;
    mbar_fence_init();
    // the first loads are under way while tensor memory is set up
    mbar_arrive_expect_tx(q_full, TILE_BYTES);
    issue_tile({smem + DQ_OFF_Q, &map_q, q0, h, b}, q_full);
    if (early) {
      mbar_arrive_expect_tx(&full[0], TILE_BYTES);
      issue_tile({smem, &map_k, j0 * 128, h, b}, &full[0]);
    }
    mbar_arrive_expect_tx(rows_full, 2 * TILE_BYTES);
    issue_tile({do_smem, &map_do, q0, h, b}, rows_full);
    issue_tile({o_smem, &map_o, q0, h, b}, rows_full);
  }
  const uint32_t tm = open_tmem(tmem_slot, warp == W::tmem);
  constexpr uint32_t T_S = 0, T_DP = 128, T_DQ = 256, T_DO = 384, T_DS = 448;

  if (warp >= W::producer) {
    other_warp_registers<ROW_WARPS_B>();
    if (warp == W::producer) {
      for (int seq = early ? 1 : 0; seq <= 2 * n; ++seq) {
        // entry 2 n: the first tile of k, for its mean
        const bool is_k = (seq & 1) == 0, mean = seq == 2 * n;
        const int j = mean ? 0 : j0 + (seq >> 1);
        const uint32_t s = seq % DQ_SLOTS, ph = (seq / DQ_SLOTS) & 1u;
        if (!mbar_wait(&empty[s], ph ^ 1u, abort_flag)) break;
        if (seq >= DQ_SLOTS - 2 && seq < DQ_SLOTS && !mbar_wait(do_full, 0, abort_flag)) break;  // do and o have been read
        const TileLoad t = {smem + s * TILE_BYTES, is_k ? &map_k : &map_v, j * 128, h, b};
        if (is_k && !mean && rem != 0 && j == n_all - 1) {
          if (!load_tile_tail(t, tail, 0, rem, &full[s], abort_flag)) break;
        } else if (lane == 0) {
          mbar_arrive_expect_tx(&full[s], TILE_BYTES);
          issue_tile(t, &full[s]);
        }
        __syncwarp();
      }
    } else if (warp == W::issuer0) {
      const bool leader = elect_one();
      const uint32_t ring = smem_u32(smem), id = idesc_k<BF16>();
      bool ok = mbar_wait(q_full, 0, abort_flag);
      for (int j = 0; ok && j < n; ++j) {
        const uint32_t ks = (2 * j) % DQ_SLOTS, kph = ((2 * j) / DQ_SLOTS) & 1u;
        const uint32_t vs = (2 * j + 1) % DQ_SLOTS, vph = ((2 * j + 1) / DQ_SLOTS) & 1u;
        ok = mbar_wait(&full[ks], kph, abort_flag) && (j == 0 || mbar_wait(s_free, (j - 1) & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          mma_ss(tm + T_S, ring + DQ_OFF_Q, ring + ks * TILE_BYTES, id);
          umma_commit(s_full);
        }
        __syncwarp();
        ok = mbar_wait(&full[vs], vph, abort_flag) && (j == 0 ? mbar_wait(do_full, 0, abort_flag) : mbar_wait(dp_free, (j - 1) & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          mma_ts_k(tm + T_DP, tm + T_DO, ring + vs * TILE_BYTES, id);
          umma_commit(dp_full);
          umma_commit(&empty[vs]);
        }
        __syncwarp();
      }
    } else if (warp == W::issuer1) {
      const bool leader = elect_one();
      const uint32_t ring = smem_u32(smem), id_mn = idesc_mn<BF16>();
      for (int j = 0; j < n; ++j) {
        const uint32_t ks = (2 * j) % DQ_SLOTS, kph = ((2 * j) / DQ_SLOTS) & 1u;
        // ds exists, so s of this tile is long complete: the slot of k is free with this product
        if (!(mbar_wait(&full[ks], kph, abort_flag) && mbar_wait(ds_full, j & 1u, abort_flag))) break;
        tc_fence_after_sync();
        if (leader) {
          mma_ts_mn(tm + T_DQ, tm + T_DS, ring + ks * TILE_BYTES, id_mn, j == 0);
          umma_commit(dq_done);
          umma_commit(&empty[ks]);
        }
        __syncwarp();
      }
    }
  } else {
    row_warp_registers<ROW_WARPS_B>();
    const int cg = warp >> 2, r = (warp & 3) * 32 + lane, q_row = q0 + r;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const bool live = q_row < q_len;
    float* s_mean = reinterpret_cast<float*>(smem + DQ_OFF_MEAN);
    const float l = live ? p.lse[static_cast<int64_t>(bh) * p.Sq + q_row] : -INFINITY;
    float v_top = 0.f;
    if constexpr (!BF16) v_top = range_of_v(p, bh);
    bool ok = mbar_wait(rows_full, 0, abort_flag);
    {  // a quarter of a row of do to tensor memory, and its part of D to where dq will be
      uint32_t w[16];
      float d[2] = {0.f, 0.f}, norm = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = (cg >> 1) * BOX_BYTES + r * 128 + ((((cg & 1) * 4 + i) ^ (r & 7)) << 4);
        uint4 u = *reinterpret_cast<const uint4*>(do_smem + at), o = *reinterpret_cast<const uint4*>(o_smem + at);
        if (!live) u = o = make_uint4(0u, 0u, 0u, 0u);
        const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, ow[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float a0, a1, o0, o1;
          unpack2<BF16>(uw[k], a0, a1);
          unpack2<BF16>(ow[k], o0, o1);
          d[0] = fmaf(a0, o0, d[0]);
          d[1] = fmaf(a1, o1, d[1]);
          if constexpr (!BF16) norm = fmaf(a0, a0, fmaf(a1, a1, norm));
          w[4 * i + k] = uw[k];
        }
      }
      tmem_st16(tm + lanes + T_DO + cg * 16, w);
      tmem_st1(tm + lanes + T_DQ + cg * 32, __float_as_uint(d[0] + d[1]));
      if constexpr (!BF16) tmem_st1(tm + lanes + T_DQ + cg * 32 + 1, __float_as_uint(norm));
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(do_full);
    }
    ok = ok && mbar_wait(do_full, 0, abort_flag);  // all warps have arrived
    tc_fence_after_sync();
    const float nl = l == -INFINITY ? -INFINITY : -l * LOG2E;
    float nd = -sum_of_groups(tm + lanes + T_DQ);
    // fp16: ds is computed and rounded times `factor`, so -D is kept times it; `to_stat` makes of that what the dk/dv kernel wants
    float factor = 1.f, to_stat = 1.f;
    if constexpr (!BF16) {
      factor = range_factor(sum_of_groups(tm + lanes + T_DQ + 1) * v_top);
      nd *= factor;
      to_stat = stat_factor(p, bh) * power_inverse(factor);
    }
    if (cg == 0 && split == 0) {
      stat[r] = nl + P_SHIFT<BF16>;
      stat[stats + r] = nd * to_stat;
    }
    const uint64_t nl2 = f2_splat(nl), cmul2 = f2_splat(p.sm_scale * LOG2E);
    uint64_t nd2 = f2_splat(nd);
    const uint64_t factor2 = f2_splat(factor);
    const auto minus_d = [factor2](uint32_t y0, uint32_t y1, uint64_t nd) {  // dp - D, times the factor
      if constexpr (BF16) return f2_add(f2_bits(y0, y1), nd);
      else return f2_fma(f2_bits(y0, y1), factor2, nd);
    };
    float e[2] = {0.f, 0.f};  // sums of the rounded ds
    const int team = warp >> 3;
    const auto tile = [&](int j, auto only) -> bool {  // the arithmetic of a tile of keys; false: a wait gave up
      const int valid = k_len - (j0 + j) * 128 - cg * 32;  // this thread's columns that exist
      if (!mbar_wait(s_full, j & 1u, abort_flag)) return false;
      tc_fence_after_sync();
      uint32_t sv[32];
      tmem_ld32(tm + lanes + T_S + cg * 32, sv);
      tmem_wait_ld();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free);
      // turn[0] opens the exponentials of team 0 (team 1 has done its last tile's), turn[1] those of team 1
      if ((team == 1 || j > 0) && !mbar_wait(&turn[team], (team == 1 ? j : j - 1) & 1u, abort_flag)) return false;
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        float a, c;
        f2_unpack(f2_fma(f2_bits(sv[i], sv[i + 1]), cmul2, nl2), a, c);
        sv[i] = __float_as_uint(ex2(a));
        sv[i + 1] = __float_as_uint(ex2(c));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&turn[team ^ 1]);
      if (!mbar_wait(dp_full, j & 1u, abort_flag)) return false;
      tc_fence_after_sync();
      uint32_t dp[32];
      tmem_ld32(tm + lanes + T_DP + cg * 32, dp);
      tmem_wait_ld();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(dp_free);
      if (valid < 32) {  // keys behind the length: whatever v holds there
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          sv[i] = i < valid ? sv[i] : 0u;
          dp[i] = i < valid ? dp[i] : 0u;
        }
      }
      if constexpr (decltype(only)::value) {  // what sum_j p (dp - D) is off zero, D is off
        uint64_t off2 = f2_splat(0.f);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          off2 = f2_fma(f2_bits(sv[2 * i], sv[2 * i + 1]), minus_d(dp[2 * i], dp[2 * i + 1], nd2), off2);
        float a, c;
        f2_unpack(off2, a, c);
        tmem_st1(tm + lanes + T_DP + cg * 32, __float_as_uint(a + c));  // where this warp has read its dp
        tmem_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(sums_full);
        if (!mbar_wait(sums_full, 0, abort_flag)) return false;
        tc_fence_after_sync();
        const float off = sum_of_groups(tm + lanes + T_DP);  // by the whole warp, rows that do not exist included
        f2_unpack(nd2, a, c);
        a = live ? a - off : 0.f;  // a row behind the length holds anything
        nd2 = f2_splat(a);
        if (cg == 0) stat[stats + r] = a * to_stat;  // split 0 has the tile
      }
      uint32_t pk[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        pk[i] = f2_to16_rn<BF16>(f2_mul(f2_bits(sv[2 * i], sv[2 * i + 1]), minus_d(dp[2 * i], dp[2 * i + 1], nd2)));
        add_pair<BF16>(e[i & 1], pk[i]);
      }
      if (j > 0) {  // ds of the last tile has been read (normally long ago)
        if (!mbar_wait(dq_done, (j - 1) & 1u, abort_flag)) return false;
        tc_fence_after_sync();
      }
      tmem_st16(tm + lanes + T_DS + cg * 16, pk);
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
      return true;
    };
    // two copies: with the sum over the row as a branch in the loop the backward pass took 2 to 3 % longer at every length
    if (n_all == 1) ok = ok && tile(0, std::true_type{});
    else
      for (int j = 0; ok && j < n; ++j) ok = tile(j, std::false_type{});
    // for the end; read (and its address computed) again instead of kept in registers over the loop
    int q_end = q0 + r;
    asm volatile("" : "+r"(q_end));
    float* stat_d = p.row_stats + (static_cast<int64_t>(p.B) * p.heads + bh) * p.Sq_pad + q_end;
    const float minus_d_stat = cg == 0 && p.splits == 1 ? *stat_d : 0.f;  // this thread's own
    if constexpr (!BF16) to_stat = stat_factor(p, bh) * power_inverse(factor);
    // m: the mean of the first tile's keys; a thread adds eight channels of four keys
    if (ok) ok = mbar_wait(&full[(2 * n) % DQ_SLOTS], ((2 * n) / DQ_SLOTS) & 1u, abort_flag);
    {
      const uint8_t* k_smem = smem + ((2 * n) % DQ_SLOTS) * TILE_BYTES;
      const int rows = min(128, k_len), chunk = threadIdx.x & 15, k0 = (threadIdx.x >> 4) * 4;
      float m[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k0 + i < rows) {
          const uint4 u = *reinterpret_cast<const uint4*>(k_smem + (chunk >> 3) * BOX_BYTES + (k0 + i) * 128 + (((chunk & 7) ^ ((k0 + i) & 7)) << 4));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float a0, a1;
            unpack2<BF16>(w[k], a0, a1);
            m[2 * k] += a0;
            m[2 * k + 1] += a1;
          }
        }
      // s of the last tile is complete (this thread has its ds): q's place is free
      const float inv = 1.f / static_cast<float>(rows);
#pragma unroll
      for (int k = 0; k < 8; ++k) m[k] = (m[k] + __shfl_xor_sync(0xffffffffu, m[k], 16)) * inv;
      if (lane < 16) {
        *reinterpret_cast<float4*>(s_mean + warp * 128 + chunk * 8) = make_float4(m[0], m[1], m[2], m[3]);
        *reinterpret_cast<float4*>(s_mean + warp * 128 + chunk * 8 + 4) = make_float4(m[4], m[5], m[6], m[7]);
      }
      tmem_st1(tm + lanes + T_S + cg * 32, __float_as_uint(e[0] + e[1]));  // the scores have all been read
      tmem_wait_st();
      tc_fence_before_sync();
      row_warps_sync();
      tc_fence_after_sync();
      if (threadIdx.x < 128) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) t += s_mean[k * 128 + threadIdx.x];
        s_mean[threadIdx.x] = t;  // only this thread reads or writes this channel until the barrier
      }
      row_warps_sync();
    }
    if (ok && mbar_wait(dq_done, (n - 1) & 1u, abort_flag)) {
      tc_fence_after_sync();
      // the softmax over one key is constant: its gradient is zero, not the rounding of dp - D
      const float unscale = BF16 ? 1.f : power_inverse(factor), mul = k_len == 1 ? 0.f : p.sm_scale * unscale;
      const float neg_e = -sum_of_groups(tm + lanes + T_S);
      if (cg == 0) {  // D + e for the dk/dv kernel (one tile of keys: e is in D already)
        const float off = live && k_len > 128 ? neg_e : 0.f;
        if (p.splits > 1) part_e()[r] = off * to_stat;
        else *stat_d = fmaf(off, to_stat, minus_d_stat);
      }
      const int rows = max(0, min(32, rows_in - (warp & 3) * 32));
      uint8_t* st = smem + warp * 4096;  // every product and every copy is complete: the ring stages the results
      uint32_t v[32];
      tmem_ld32(tm + lanes + T_DQ + cg * 32, v);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const float4 m = *reinterpret_cast<const float4*>(s_mean + cg * 32 + i);
        v[i] = __float_as_uint(fmaf(neg_e, m.x, __uint_as_float(v[i])));
        v[i + 1] = __float_as_uint(fmaf(neg_e, m.y, __uint_as_float(v[i + 1])));
        v[i + 2] = __float_as_uint(fmaf(neg_e, m.z, __uint_as_float(v[i + 2])));
        v[i + 3] = __float_as_uint(fmaf(neg_e, m.w, __uint_as_float(v[i + 3])));
      }
      if (p.splits > 1) store_part32(st, v, unscale, live, part + (warp & 3) * 32 * 128 + cg * 32, rows);
      else store_cols32<BF16>(st, v, mul, live, out_ptr(p.dq, b, h, q0 + (warp & 3) * 32) + cg * 32, p.dq.st, rows);
    }
  }
  close_tmem(tm, warp == W::tmem, abort_flag, p.status);
}

// ---- dk, dv ------------------------------------------------------------------------------------------------------------
// One CTA = 128 keys of one head; k and v stay in shared memory, q and do tiles pass through the ring.  Everything is
// transposed: a thread owns a KEY row x 32 queries, so p^T and ds^T come out as A operands of dv += p^T.do and
// dk += ds^T.q and never leave tensor memory; lse and D of the queries are read along the row.
//   issuer 0     s^T = k.q_i^T and dp^T = v.do_i^T        issuer 1     dv += p^T.do_i and dk += ds^T.q_i
// Tensor memory: s^T, then dp^T in the same place [0,128)   p^T [128,192)   ds^T [192,256)   dv [256,384)   dk [384,512): all
// of it.  s^T and dp^T are free as soon as they are in registers: dp^T is computed under the exponentials, s^T of the next
// tile under the arithmetic of ds^T, and neither waits for a product that reads p^T or ds^T.  Those are handed over in
// halves, so that the first half's product runs under the second half's arithmetic.
// 8 heads x 4,096 x 4,096 bf16: 133 us (138 with p^T over s^T and ds^T over dp^T, where s^T of the next tile has to wait for
// dv); a tile takes 2,800 clocks: 1,260 for the exponentials (the unit's own time is 1,024), 740 for ds^T, the rest waits for
// products and loads.  The four products alone take 2,048 (tensor pipe 64 %).
constexpr int KV_SLOTS = 4;
constexpr int KV_OFF_K = KV_SLOTS * TILE_BYTES;
constexpr int KV_OFF_V = KV_OFF_K + TILE_BYTES;
constexpr int KV_OFF_STAT = KV_OFF_V + TILE_BYTES;  // [2 stages][2][128] floats
constexpr int KV_OFF_BAR = KV_OFF_STAT + 2048;
constexpr int KV_SMEM = KV_OFF_BAR + 256 + 1024;

template <bool BF16>
__global__ void __launch_bounds__(Warps<ROW_WARPS_B>::threads, 1)
attn_bwd_dkdv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                     const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TrainParams p) {
  using W = Warps<ROW_WARPS_B>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k0 = blockIdx.x * 128, bh = blockIdx.y, b = bh / p.heads, h = bh % p.heads, split = blockIdx.z;
  const int q_len = valid_len(p.q_lens, b, p.Sq), k_len = valid_len(p.k_lens, b, p.Sk);
  const int n_all = k0 < k_len ? (q_len + 127) / 128 : 0;
  const int per = (n_all + p.splits - 1) / p.splits;
  const int i0 = split * per, n = max(0, min(n_all, i0 + per) - i0);
  // a split run leaves fp32 sums: dk [split][BH][Sk][128], then dv the same
  const int64_t part_all = static_cast<int64_t>(p.splits) * p.B * p.heads * p.Sk * 128;
  float* part = p.part + ((static_cast<int64_t>(split) * p.B * p.heads + bh) * p.Sk + k0) * 128;
  const int rows_in = min(128, p.Sk - k0);

  if (n == 0) {
    if (p.splits > 1) {
      zero_rows(part, 512, rows_in, 512);
      zero_rows(part + part_all, 512, rows_in, 512);
    } else {
      zero_rows(out_ptr(p.dk, b, h, k0), p.dk.st * 2, rows_in, 256);
      zero_rows(out_ptr(p.dv, b, h, k0), p.dv.st * 2, rows_in, 256);
    }
    return;
  }

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + KV_OFF_BAR);
  uint64_t* full = bars;                // [KV_SLOTS]
  uint64_t* empty = full + KV_SLOTS;    // [KV_SLOTS] released by the two products that read the tile
  uint64_t* tail = empty + KV_SLOTS;
  uint64_t* k_full = tail + 1;
  uint64_t* v_full = k_full + 1;
  uint64_t* s_full = v_full + 1;
  uint64_t* s_free = s_full + 1;
  uint64_t* p_full = s_free + 1;        // [2] halves of every thread's queries
  uint64_t* dv_done = p_full + 2;
  uint64_t* dp_full = dv_done + 1;
  uint64_t* dp_free = dp_full + 1;
  uint64_t* ds_full = dp_free + 1;      // [2]
  uint64_t* dk_done = ds_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dk_done + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  if (warp == W::producer && lane == 0) {
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_v);
    tma_prefetch_desc(&map_do);
    for (int i = 0; i < KV_SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 2);
    }
    mbar_init(tail, 1);
    mbar_init(k_full, 1);
    mbar_init(v_full, 1);
    mbar_init(s_full, 1);
    mbar_init(s_free, ROW_WARPS_B);
    mbar_init(dv_done, 1);
    mbar_init(dp_full, 1);
    mbar_init(dp_free, ROW_WARPS_B);
    mbar_init(dk_done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&p_full[i], ROW_WARPS_B);
      mbar_init(&ds_full[i], ROW_WARPS_B);
    }
    *abort_flag = 0;
    mbar_fence_init();
    // the first loads are under way while tensor memory is set up
    mbar_arrive_expect_tx(k_full, TILE_BYTES);
    issue_tile({smem + KV_OFF_K, &map_k, k0, h, b}, k_full);
    mbar_arrive_expect_tx(v_full, TILE_BYTES);
    issue_tile({smem + KV_OFF_V, &map_v, k0, h, b}, v_full);
  }
  const uint32_t tm = open_tmem(tmem_slot, warp == W::tmem);
  constexpr uint32_t T_S = 0, T_P = 128, T_DS = 192, T_DV = 256, T_DK = 384;
  const int64_t stats = static_cast<int64_t>(p.B) * p.heads * p.Sq_pad;

  if (warp >= W::producer) {
    other_warp_registers<ROW_WARPS_B>();
    if (warp == W::producer) {
      const int rem = q_len < p.Sq ? q_len % 128 : 0;
      for (int seq = 0; seq < 2 * n; ++seq) {
        const int i = i0 + (seq >> 1);
        const uint32_t s = seq % KV_SLOTS, ph = (seq / KV_SLOTS) & 1u;
        if (!mbar_wait(&empty[s], ph ^ 1u, abort_flag)) break;
        const bool is_q = (seq & 1) == 0, clear = rem != 0 && i == n_all - 1;
        const TileLoad t = {smem + s * TILE_BYTES, is_q ? &map_q : &map_do, i * 128, h, b};
        if (lane == 0) {
          // lse and D of the tile's queries ride on the q tile's barrier; the stage is free with the slot.  Where a tail is
          // cleared, the arrival (and the tile's own bytes) are load_tile_tail's
          if (!clear) mbar_arrive_expect_tx(&full[s], TILE_BYTES + (is_q ? 1024u : 0u));
          else if (is_q) mbar_expect_tx(&full[s], 1024u);
          if (is_q) {
            float* dst = reinterpret_cast<float*>(smem + KV_OFF_STAT) + (seq / 2 % 2) * 256;
            const float* src = p.row_stats + static_cast<int64_t>(bh) * p.Sq_pad + i * 128;
            bulk_load(dst, src, 512, &full[s]);
            bulk_load(dst + 128, src + stats, 512, &full[s]);
          }
          if (!clear) issue_tile(t, &full[s]);
        }
        __syncwarp();
        if (clear && !load_tile_tail(t, tail, is_q ? 0u : 1u, rem, &full[s], abort_flag)) break;
      }
    } else if (warp == W::issuer0) {
      const bool leader = elect_one();
      const uint32_t ring = smem_u32(smem), id = idesc_k<BF16>();
      bool ok = mbar_wait(k_full, 0, abort_flag);
      for (int i = 0; ok && i < n; ++i) {
        const uint32_t seq = 2 * i, s = seq % KV_SLOTS, ph = (seq / KV_SLOTS) & 1u, s1 = (seq + 1) % KV_SLOTS, ph1 = ((seq + 1) / KV_SLOTS) & 1u;
        ok = mbar_wait(&full[s], ph, abort_flag) && (i == 0 || mbar_wait(dp_free, (i - 1) & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          mma_ss(tm + T_S, ring + KV_OFF_K, ring + s * TILE_BYTES, id);
          umma_commit(s_full);
          umma_commit(&empty[s]);
        }
        __syncwarp();
        ok = (i > 0 || mbar_wait(v_full, 0, abort_flag)) && mbar_wait(&full[s1], ph1, abort_flag) && mbar_wait(s_free, i & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after_sync();
        if (leader) {
          mma_ss(tm + T_S, ring + KV_OFF_V, ring + s1 * TILE_BYTES, id);
          umma_commit(dp_full);
          umma_commit(&empty[s1]);
        }
        __syncwarp();
      }
    } else if (warp == W::issuer1) {
      const bool leader = elect_one();
      const uint32_t ring = smem_u32(smem), id_mn = idesc_mn<BF16>();
      bool ok = true;
      for (int i = 0; ok && i < n; ++i) {
        const uint32_t seq = 2 * i, s = seq % KV_SLOTS, ph = (seq / KV_SLOTS) & 1u, s1 = (seq + 1) % KV_SLOTS, ph1 = ((seq + 1) / KV_SLOTS) & 1u;
        ok = mbar_wait(&full[s1], ph1, abort_flag);
        for (int c = 0; ok && c < 2; ++c) {
          if (!(ok = mbar_wait(&p_full[c], i & 1u, abort_flag))) break;
          tc_fence_after_sync();
          if (leader) mma_ts_mn_half(tm + T_DV, tm + T_P, c, ring + s1 * TILE_BYTES, id_mn, i == 0 && c == 0);
          __syncwarp();
        }
        if (!ok) break;
        if (leader) {
          umma_commit(dv_done);
          umma_commit(&empty[s1]);
        }
        __syncwarp();
        ok = mbar_wait(&full[s], ph, abort_flag);
        for (int c = 0; ok && c < 2; ++c) {
          if (!(ok = mbar_wait(&ds_full[c], i & 1u, abort_flag))) break;
          tc_fence_after_sync();
          if (leader) mma_ts_mn_half(tm + T_DK, tm + T_DS, c, ring + s * TILE_BYTES, id_mn, i == 0 && c == 0);
          __syncwarp();
        }
        if (!ok) break;
        if (leader) {
          umma_commit(dk_done);
          umma_commit(&empty[s]);
        }
        __syncwarp();
      }
    }
  } else {
    row_warp_registers<ROW_WARPS_B>();
    const int cg = warp >> 2, k_row = k0 + (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint64_t cmul2 = f2_splat(p.sm_scale * LOG2E);
    // fp16: 2^P_SHIFT p is at hand and the head's factor times ds is wanted (-D comes with both in it)
    float unscale = 1.f, factor = 1.f;
    if constexpr (!BF16) {
      factor = stat_factor(p, bh);
      unscale = P_UNSHIFT<BF16> * power_inverse(factor);
    }
    const uint64_t factor2 = f2_splat(factor);
    const auto minus_d = [factor2](uint32_t y0, uint32_t y1, uint64_t nd) {
      if constexpr (BF16) return f2_add(f2_bits(y0, y1), nd);
      else return f2_fma(f2_bits(y0, y1), factor2, nd);
    };
    bool ok = true;
    for (int i = 0; ok && i < n; ++i) {
      const ulonglong2* stat = reinterpret_cast<const ulonglong2*>(smem + KV_OFF_STAT + (i % 2) * 1024 + cg * 128);  // four queries each
      const uint32_t seq = 2 * i;
      ok = mbar_wait(&full[seq % KV_SLOTS], (seq / KV_SLOTS) & 1u, abort_flag) && mbar_wait(s_full, i & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after_sync();
      uint32_t sv[32];
      tmem_ld32(tm + lanes + T_S + cg * 32, sv);
      tmem_wait_ld();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t pk[8];
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
          const ulonglong2 nl = stat[4 * c + k / 4];
          uint32_t* x = &sv[16 * c + k];
          float a0, a1, a2, a3;
          f2_unpack(f2_fma(f2_bits(x[0], x[1]), cmul2, nl.x), a0, a1);
          f2_unpack(f2_fma(f2_bits(x[2], x[3]), cmul2, nl.y), a2, a3);
          a0 = ex2(a0);
          a1 = ex2(a1);
          a2 = ex2(a2);
          a3 = ex2(a3);
          x[0] = __float_as_uint(a0);
          x[1] = __float_as_uint(a1);
          x[2] = __float_as_uint(a2);
          x[3] = __float_as_uint(a3);
          pk[k / 2] = pack2_rn<BF16>(a0, a1);
          pk[k / 2 + 1] = pack2_rn<BF16>(a2, a3);
        }
        if (c == 0 && i > 0) {  // p of the last tile has been read (normally long ago)
          if (!(ok = mbar_wait(dv_done, (i - 1) & 1u, abort_flag))) break;
          tc_fence_after_sync();
        }
        tmem_st8(tm + lanes + T_P + cg * 16 + 8 * c, pk);
        tmem_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[c]);
      }
      if (!ok || !(ok = mbar_wait(dp_full, i & 1u, abort_flag))) break;
      tc_fence_after_sync();
      uint32_t dp[32];
      tmem_ld32(tm + lanes + T_S + cg * 32, dp);
      tmem_wait_ld();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(dp_free);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t pk[8];
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
          const ulonglong2 nd = stat[32 + 4 * c + k / 4];
          const uint32_t* x = &sv[16 * c + k];
          const uint32_t* y = &dp[16 * c + k];
          pk[k / 2] = f2_to16_rn<BF16>(f2_mul(f2_bits(x[0], x[1]), minus_d(y[0], y[1], nd.x)));
          pk[k / 2 + 1] = f2_to16_rn<BF16>(f2_mul(f2_bits(x[2], x[3]), minus_d(y[2], y[3], nd.y)));
        }
        if (c == 0 && i > 0) {  // and so has ds
          if (!(ok = mbar_wait(dk_done, (i - 1) & 1u, abort_flag))) break;
          tc_fence_after_sync();
        }
        tmem_st8(tm + lanes + T_DS + cg * 16 + 8 * c, pk);
        tmem_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_full[c]);
      }
    }
    if (ok && mbar_wait(dv_done, (n - 1) & 1u, abort_flag) && mbar_wait(dk_done, (n - 1) & 1u, abort_flag)) {
      tc_fence_after_sync();
      const bool live = k_row < k_len;
      const float mul = k_len == 1 ? 0.f : p.sm_scale * unscale;  // one key: see the dq kernel
      const int row0 = (warp & 3) * 32, rows = max(0, min(32, rows_in - row0));
      uint8_t* st = smem + warp * 4096;  // every product and every copy is complete: the ring stages the results
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        uint32_t v[32];
        tmem_ld32(tm + lanes + (c == 0 ? T_DK : T_DV) + cg * 32, v);
        tmem_wait_ld();
        if (p.splits > 1) store_part32(st, v, c == 0 ? unscale : P_UNSHIFT<BF16>, live, part + (c == 0 ? 0 : part_all) + row0 * 128 + cg * 32, rows);
        else store_cols32<BF16>(st, v, c == 0 ? mul : P_UNSHIFT<BF16>, live, out_ptr(c == 0 ? p.dk : p.dv, b, h, k0 + row0) + cg * 32, (c == 0 ? p.dk : p.dv).st, rows);
      }
    }
  }
  close_tmem(tm, warp == W::tmem, abort_flag, p.status);
}

// ---- forward -----------------------------------------------------------------------------------------------------------
// The schedule of attn_fwd_tmem_p_kernel (attn_tmem.cu: 256 query rows per CTA as two tiles, one shared score buffer,
// probabilities through tensor memory, five-slot ring of k and v tiles) with what training asks of it: lengths, fp16,
// any strides, the log-sum-exp, probabilities rounded instead of truncated, and, where there are too few rows to fill the
// GPU, the keys split over several CTAs.  8 heads x 4,096 x 4,096 bf16: 64 us, tensor pipe 69 %, unit of the exponentials 70 %.
constexpr int F_SLOTS = 5;
constexpr int F_OFF_Q = 0;
constexpr int F_OFF_RING = 2 * TILE_BYTES;
constexpr int F_OFF_BAR = F_OFF_RING + F_SLOTS * TILE_BYTES;
constexpr int F_SMEM = F_OFF_BAR + 256 + 1024;

template <bool BF16>
__global__ void __launch_bounds__(Warps<ROW_WARPS_F>::threads, 1)
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
  const int rows_in = max(0, min(256, p.Sq - q0));  // rows of the CTA
  if (n == 0) {  // zeros, or a part of zero weight
    if (p.splits > 1) {
      float* part = p.part + (static_cast<int64_t>(split) * p.B * p.heads * p.Sq + static_cast<int64_t>(bh) * p.Sq + q0) * 128;
      zero_rows(part, 512, rows_in, 512);
      if (warp < 8 && q_row < p.Sq) p.part_lse[split_row] = -INFINITY;
    } else {
      zero_rows(out_ptr(p.o, b, h, q0), p.o.st * 2, rows_in, 256);
      if (warp < 8 && q_row < p.Sq) p.lse[row] = -INFINITY;
    }
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
  using W = Warps<ROW_WARPS_F>;
  const int rem = k_len < p.Sk ? k_len % 128 : 0;  // tokens of the last tile that exist (0: no tail of v to clear)
  if (warp == W::producer && lane == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
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
    // the first loads are under way while tensor memory is set up
    mbar_arrive_expect_tx(q_full, tiles * TILE_BYTES);
    for (int t = 0; t < tiles; ++t) issue_tile({smem + F_OFF_Q + t * TILE_BYTES, &map_q, q0 + t * 128, h, b}, q_full);
    mbar_arrive_expect_tx(&kv_full[0], TILE_BYTES);
    issue_tile({smem + F_OFF_RING, &map_k, j0 * 128, h, b}, &kv_full[0]);
  }
  const uint32_t tm = open_tmem(tmem_slot, warp == W::tmem);

  if (warp >= W::producer) {
    other_warp_registers<ROW_WARPS_F>();
    if (warp == W::producer) {
      for (int seq = 1; seq < 2 * n; ++seq) {
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
    } else if (warp == W::issuer0) {
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
    } else if (warp == W::issuer1) {
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
          mma_ts_mn(tm + 256 + t * 128, tm + 128 + t * 64, ring + s * TILE_BYTES, id_mn, j == 0);
          umma_commit(&pv_done[t]);
          umma_commit(&kv_empty[s]);
        }
        __syncwarp();
      }
    }
  } else if (x < tiles) {
    row_warp_registers<ROW_WARPS_F>();
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
      const float m_new = (mx > m + TAU<BF16>) ? mx : m;
      const float alpha = ex2(m - m_new);  // m = -inf on the first tile -> 0
      const float off = F_SHIFT<BF16> - m_new;
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
          pk[c] = pack2_rn<BF16>(e0, e1);
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
      const float inv_l = 1.f / l, l2 = m + (log2f(l) - F_SHIFT<BF16>);
      if (q_row < p.Sq) (p.splits > 1 ? p.part_lse[split_row] : p.lse[row]) = live ? (p.splits > 1 ? l2 : l2 * LN2) : -INFINITY;
      // the tile's scores are complete, so its q has been read for the last time: its place stages the results
      uint8_t* st = smem + F_OFF_Q + x * TILE_BYTES + (warp & 3) * 8192;
      const int row0 = q_row - lane, rows = max(0, min(32, p.Sq - row0));
      float* part = p.part + (split_row - lane) * 128;
      uint16_t* dst = out_ptr(p.o, b, h, row0);
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t ov[32];
        tmem_ld32(o_tmem + c * 32, ov);
        tmem_wait_ld();
        if (p.splits > 1) store_part32(st, ov, inv_l, live, part + 32 * c, rows);
        else store_cols32<BF16>(st, ov, inv_l, live, dst + 32 * c, p.o.st, rows);
      }
    }
  } else {  // a second tile without rows that exist: zeros for those of the tensor
    other_warp_registers<ROW_WARPS_F>();
    const int row0 = q_row - lane, rows = max(0, min(32, p.Sq - row0));
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    for (int i = 0; i < rows; ++i) {
      if (p.splits > 1) *reinterpret_cast<uint4*>(p.part + (split_row - lane + i) * 128 + lane * 4) = z;
      else if (lane < 16) *reinterpret_cast<uint4*>(out_ptr(p.o, b, h, row0 + i) + lane * 8) = z;
    }
    if (lane < rows) (p.splits > 1 ? p.part_lse[split_row] : p.lse[row]) = -INFINITY;
  }
  close_tmem(tm, warp == W::tmem, abort_flag, p.status);
}

// ---- joins of split runs -------------------------------------------------------------------------------------------------
// One thread = four channels of a row; the parts are added in the order of the splits.
template <bool BF16>
__device__ __forceinline__ void store4(uint16_t* dst, float4 v, float mul) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack2_rn<BF16>(v.x * mul, v.y * mul), pack2_rn<BF16>(v.z * mul, v.w * mul));
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

struct JoinTarget {
  Rows out;
  const float* part;
  const int* k_lens;
  float mul;
  bool scores;  // dq, dk: a gradient through the scores, zero where there is one key only
  const float* part_e;  // dq: its parts of the rows' e ...
  float* stat;          // ... and -D, which takes their sum: [BH, Sq_pad]
  int S_pad;
};
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
  const float mul = t.scores && valid_len(t.k_lens, b, Sk) == 1 ? 0.f : t.mul;
  store4<BF16>(out_ptr(t.out, b, bh % heads, s) + c, acc, mul);
  if (t.stat != nullptr && c == 0) {
    const int64_t at = static_cast<int64_t>(bh) * t.S_pad + s, stride = rows / S * t.S_pad;
    float off = 0.f;
    for (int k = 0; k < splits; ++k) off += t.part_e[k * stride + at];
    t.stat[at] += off;
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// Splits of the long axis.  `units` CTAs walk over `inner` tiles each; they run in waves of one CTA per SM, so a launch takes
// waves x (tiles per CTA + `fixed`), `fixed` being the prologue and epilogue of a CTA in tiles.  Splitting fills the last
// wave and, with few rows, the GPU, but costs another launch and its fp32 parts are written and read again: `join` tiles'
// time for a whole wave's parts (forward: 2 x 132 KB per CTA at 5 TB/s against 1.6 us per tile).
// Measured, us, forward and backward, whole / split by this rule: 8 queries x 30,000 keys 276 and 279 / 41 and 54;
// 30,000 x 100 31 and 376 / 32 and 63; 4 heads x 1,024 x 8,192 104 and 125 / 41 and 81; 5 heads x 8,190 206 and 551 / 195
// and 558 (the estimate is off by a per cent there); 12 x 4,095 and 20 x 1,560 stay whole.
inline int choose_splits(int64_t units, int64_t inner, double fixed, double join) {
  const int64_t sms = sm_count();
  int best = 1;
  double best_cost = 0;
  for (int s = 1; s <= kMaxSplits && (s == 1 || inner >= 2 * s); ++s) {
    const double waves = static_cast<double>((units * s + sms - 1) / sms);
    const double cost = waves * (static_cast<double>((inner + s - 1) / s) + fixed) + (s > 1 ? 3.0 + join * static_cast<double>(units * s) / sms : 0.0);
    if (s == 1 || cost < 0.97 * best_cost) {
      best = s;
      best_cost = cost;
    }
  }
  return best;
}
inline int64_t tiles_of(int64_t S, int64_t t) { return (S + t - 1) / t; }
inline int forward_splits(int64_t BH, int64_t Sq, int64_t Sk) { return choose_splits(BH * tiles_of(Sq, 256), tiles_of(Sk, 128), 3.0, 5.0); }
inline int dq_splits(int64_t BH, int64_t Sq, int64_t Sk) { return choose_splits(BH * tiles_of(Sq, 128), tiles_of(Sk, 128), 5.0, 3.0); }
inline int dkdv_splits(int64_t BH, int64_t Sq, int64_t Sk) { return choose_splits(BH * tiles_of(Sk, 128), tiles_of(Sq, 128), 4.0, 4.0); }
inline int64_t pad128(int64_t S) { return tiles_of(S, 128) * 128; }
inline size_t round256(size_t n) { return (n + 255) / 256 * 256; }

struct BackwardLayout { size_t stats, range, e, dq, dkdv, bytes; };
inline BackwardLayout backward_layout(int64_t BH, int64_t Sq, int64_t Sk) {
  BackwardLayout w{};
  const int s_q = dq_splits(BH, Sq, Sk), s_kv = dkdv_splits(BH, Sq, Sk);
  w.stats = 0;
  w.range = round256(static_cast<size_t>(BH) * pad128(Sq) * 8);
  w.e = w.range + round256(static_cast<size_t>(BH) * kRangeChunks * 8);
  w.dq = w.e + (s_q > 1 ? round256(static_cast<size_t>(s_q) * BH * pad128(Sq) * 4) : 0);
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

// The shared-memory limit of a kernel is set once per device (concurrent first calls set the same value).
template <typename K, K kernel>
int allow_smem(int bytes) {
  static std::atomic<bool> done[64] = {};
  int dev = 0;
  DAX_CUDA(cudaGetDevice(&dev));
  if (dev < 64 && done[dev].load(std::memory_order_relaxed)) return DAX_OK;
  DAX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) done[dev].store(true, std::memory_order_relaxed);
  return DAX_OK;
}

#define DAX_TRY(expr)              \
  do {                             \
    const int rc__ = (expr);       \
    if (rc__ != DAX_OK) return rc__; \
  } while (0)

template <bool BF16>
int run_forward(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const TrainParams& p, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(tiles_of(p.Sq, 256)), static_cast<unsigned>(p.B * p.heads), static_cast<unsigned>(p.splits));
  DAX_TRY((allow_smem<decltype(&attn_fwd_lse_kernel<BF16>), &attn_fwd_lse_kernel<BF16>>(F_SMEM)));
  attn_fwd_lse_kernel<BF16><<<grid, Warps<ROW_WARPS_F>::threads, F_SMEM, st>>>(mq, mk, mv, p);
  DAX_CUDA(cudaGetLastError());
  if (p.splits > 1) {
    attn_fwd_join_kernel<BF16><<<static_cast<unsigned>(tiles_of(static_cast<int64_t>(p.B) * p.heads * p.Sq, 8)), 256, 0, st>>>(p);
    DAX_CUDA(cudaGetLastError());
  }
  return DAX_OK;
}

template <bool BF16>
int run_backward(const CUtensorMap& mq, const CUtensorMap& mdo, const CUtensorMap& mo, const CUtensorMap& mk, const CUtensorMap& mv, const Rows& v,
                 const Rows& dout, TrainParams p, int s_q, int s_kv, float* part_q, float* part_kv, cudaStream_t st) {
  const unsigned BH = static_cast<unsigned>(p.B * p.heads);
  if constexpr (!BF16) {
    const int chunks = std::max((p.Sq + range_rows(p.Sq) - 1) / range_rows(p.Sq), (p.Sk + range_rows(p.Sk) - 1) / range_rows(p.Sk));
    attn_range_kernel<<<dim3(static_cast<unsigned>(chunks), BH, 2), 256, 0, st>>>(v, dout, p);
    DAX_CUDA(cudaGetLastError());
  }
  p.splits = s_q;
  p.part = part_q;
  DAX_TRY((allow_smem<decltype(&attn_bwd_dq_kernel<BF16>), &attn_bwd_dq_kernel<BF16>>(DQ_SMEM)));
  attn_bwd_dq_kernel<BF16><<<dim3(static_cast<unsigned>(tiles_of(p.Sq, 128)), BH, static_cast<unsigned>(s_q)), Warps<ROW_WARPS_B>::threads, DQ_SMEM, st>>>(mq, mdo, mo, mk, mv, p);
  DAX_CUDA(cudaGetLastError());
  if (s_q > 1) {
    const int64_t rows = static_cast<int64_t>(BH) * p.Sq;
    const JoinTarget t = {p.dq, part_q, p.k_lens, p.sm_scale, true, p.part_e, p.row_stats + static_cast<int64_t>(BH) * p.Sq_pad, p.Sq_pad};
    attn_bwd_join_kernel<BF16><<<dim3(static_cast<unsigned>(tiles_of(rows, 8)), 1), 256, 0, st>>>(t, t, s_q, rows, p.Sq, p.heads, p.Sk);
    DAX_CUDA(cudaGetLastError());
  }
  if (p.dk.p == nullptr) return DAX_OK;  // neither dk nor dv is wanted
  p.splits = s_kv;
  p.part = part_kv;
  DAX_TRY((allow_smem<decltype(&attn_bwd_dkdv_kernel<BF16>), &attn_bwd_dkdv_kernel<BF16>>(KV_SMEM)));
  attn_bwd_dkdv_kernel<BF16><<<dim3(static_cast<unsigned>(tiles_of(p.Sk, 128)), BH, static_cast<unsigned>(s_kv)), Warps<ROW_WARPS_B>::threads, KV_SMEM, st>>>(mq, mdo, mk, mv, p);
  DAX_CUDA(cudaGetLastError());
  if (s_kv > 1) {
    const int64_t rows = static_cast<int64_t>(BH) * p.Sk;
    const JoinTarget tk = {p.dk, part_kv, p.k_lens, p.sm_scale, true, nullptr, nullptr, 0},
                     tv = {p.dv, part_kv + s_kv * rows * 128, p.k_lens, 1.f, false, nullptr, nullptr, 0};
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

int dax_attn_lse_kernels(int64_t B, int64_t heads, int64_t Sq, int64_t Sk) {
  if (B <= 0 || heads <= 0 || Sq <= 0 || Sk <= 0) return 0;
  return dax::forward_splits(B * heads, Sq, Sk) > 1 ? 2 : 1;
}

int dax_attn_backward_kernels(int dtype, int64_t B, int64_t heads, int64_t Sq, int64_t Sk, int keys) {
  using namespace dax;
  if (B <= 0 || heads <= 0 || Sq <= 0 || Sk <= 0) return 0;
  return (dtype == DAX_F16 ? 1 : 0) + (dq_splits(B * heads, Sq, Sk) > 1 ? 2 : 1) + (keys == 0 ? 0 : dkdv_splits(B * heads, Sq, Sk) > 1 ? 2 : 1);
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
  const bool keys = dk != nullptr || dv != nullptr;
  if (keys) {
    DAX_TRY(check_rows(what, "dk", dk, dk_strides));
    DAX_TRY(check_rows(what, "dv", dv, dv_strides));
  }
  DAX_REQUIRE(lse != nullptr, DAX_ERR_INVALID, "%s: lse is null", what);
  const BackwardLayout w = backward_layout(B * heads, Sq, Sk);
  DAX_REQUIRE(workspace != nullptr && workspace_bytes >= w.bytes, DAX_ERR_INVALID,
              "%s: workspace of %zu bytes is smaller than the %zu required", what, workspace_bytes, w.bytes);
  DAX_REQUIRE(aligned16(workspace), DAX_ERR_ALIGN, "%s: workspace must be 16-byte aligned", what);
  CUtensorMap mq, mdo, mo, mk, mv;
  DAX_TRY(make_map(&mq, q, q_strides, Sq, heads, B));
  DAX_TRY(make_map(&mdo, dout, do_strides, Sq, heads, B));
  DAX_TRY(make_map(&mo, o, o_strides, Sq, heads, B));
  DAX_TRY(make_map(&mk, k, k_strides, Sk, heads, B));
  DAX_TRY(make_map(&mv, v, v_strides, Sk, heads, B));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  TrainParams p{};
  p.dq = rows_of(dq, dq_strides);
  if (keys) {
    p.dk = rows_of(dk, dk_strides);
    p.dv = rows_of(dv, dv_strides);
  }
  p.lse = const_cast<float*>(lse);
  p.q_lens = q_lens;
  p.k_lens = k_lens;
  p.row_stats = reinterpret_cast<float*>(ws + w.stats);
  p.range = reinterpret_cast<float*>(ws + w.range);
  p.part_e = reinterpret_cast<float*>(ws + w.e);
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
  const Rows rv = rows_of(v, v_strides), rdo = rows_of(dout, do_strides);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == DAX_BF16 ? run_backward<true>(mq, mdo, mo, mk, mv, rv, rdo, p, s_q, s_kv, part_q, part_kv, st)
                           : run_backward<false>(mq, mdo, mo, mk, mv, rv, rdo, p, s_q, s_kv, part_q, part_kv, st);
}

}  // extern "C"
