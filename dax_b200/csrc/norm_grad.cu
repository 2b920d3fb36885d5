// The row-wise steps of a DiT block for training: LayerNorm with adaLN modulation and RMSNorm with rotary embedding,
// forward (keeping the row statistics) and backward (with the column sums that are the gradients of the per-channel
// vectors).  Rows are x[b, s, :] of a [B, S, D] tensor; n is the normalised row.
//
//   LayerNorm   n = (x - mean) rstd      y = (n w + c) (1 + scale_b) + shift_b
//               g = dy (1 + scale_b) w   dx = rstd (g - mean(g) - n mean(g n))
//               A_b = sum_s dy, N_b = sum_s dy n:   dshift_b = A_b, dscale_b = w N_b + c A_b,
//               dw = sum_b (1 + scale_b) N_b, dc = sum_b (1 + scale_b) A_b
//   RMSNorm     n = x rstd               y = R_s (n w)   (R_s rotates channel pairs by the angles of table row s)
//               h = R_s^T dy, g = h w    dx = rstd (g - n mean(g n)),   dw = sum_{b, s} h n
//
// Bound by HBM: the forward pass reads x and writes y, the backward pass reads x and dy and writes dx, each once.  One
// CTA owns one or two rows at a time and walks over the rows of one sample; a thread owns the same 16-byte pieces of every
// row, so
//  - the rows travel through a ring in shared memory that each thread fills (cp.async) and reads back for itself: the
//    bytes in flight cost neither registers nor barriers.  The backward pass reads a row from there twice, before and after
//    its sums, because the registers are full of column sums;
//  - the column sums over the CTA's rows stay in the thread's registers (fp32, rows in a fixed order) and reach memory
//    once per CTA; a second kernel adds the CTAs' partial sums in a fixed order, so results do not depend on timing.
// What a row costs beside its bytes is the wait for its sums (shuffles, one barrier): two rows share one where registers and
// shared memory allow, and two to four CTAs per SM fill each other's waits.
// Statistics, coefficients and sums are fp32; y and dx are rounded once, when they are stored.
//
// Measured (x and y, or x, dy and dx, once each, each pass on its own, replayed from a graph; a plain copy reaches 6.5 TB/s),
// us forward and backward with its sums: 32,760 x 5,120 bf16 LayerNorm + modulation 118 (5.7 TB/s) and 183 (5.5), RMSNorm +
// rotation 109 (6.2) and 204 (4.9), fp16 118 and 207, 109 and 211; 16,380 x 5,120 fp32 124 (5.4) and 183 (5.5), 120 (5.6) and 189 (5.3);
// 2 x 4,095 x 1,536 fp16 affine LayerNorm 12 and 27.  What is left beside the bytes is issue slots (58 % used in the backward pass, two rounds over a row
// that lives in shared memory) and the waits for a row's sums.
#include <algorithm>
#include <atomic>

#include "quant_common.cuh"

namespace dax {
namespace {

constexpr int64_t kMaxWidth = 8192;
constexpr int kMaxSmem = 220 * 1024;  // of a CTA; the widest fp32 rows take 160 KB

struct NormArgs {
  const uint8_t* x;       // input rows
  const uint8_t* dy;      // backward: gradient rows
  uint8_t* out;           // y (forward) or dx (backward)
  int64_t x_sb, x_ss, dy_sb, dy_ss, out_sb, out_ss;  // byte strides: sample, token
  const float* weight;    // [D] or null (1)
  const float* bias;      // [D] or null (0)
  const float* shift;     // [B, D] or null (0)
  const float* scale;     // [B, D] or null (0)
  const float* cos;       // [S, 64] or null (no rotation)
  const float* sin;
  float* mean;            // [B, S] statistics: written forward, read backward (LayerNorm)
  float* rstd;            // [B, S]
  float* part;            // backward: [B, gridDim.x, SUMS, D] column sums
  int64_t S;
  int D;
  float eps;
};

// 16 bytes, or 16 zero bytes where there is nothing to read (then the address is not used)
__device__ __forceinline__ void cp_async16(void* smem_dst, const void* gmem_src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(smem_dst))),
               "l"(gmem_src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ---- 16-byte pieces: eight 16-bit or four fp32 elements ------------------------------------------------------------
template <int DT> struct Piece { static constexpr int value = DT == DAX_F32 ? 4 : 8; };

// All arithmetic runs on fp32 pairs: the kernels are closer to the bound of instruction issue than the bytes suggest.
template <int DT> struct Pairs { uint64_t v[Piece<DT>::value / 2]; };
template <int DT>
__device__ __forceinline__ Pairs<DT> unpack(const uint4& r) {
  Pairs<DT> f;
  if constexpr (DT == DAX_F32) {
    f.v[0] = f2_pack(__uint_as_float(r.x), __uint_as_float(r.y));
    f.v[1] = f2_pack(__uint_as_float(r.z), __uint_as_float(r.w));
  } else {
    f.v[0] = f2_from16<DT == DAX_BF16>(r.x);
    f.v[1] = f2_from16<DT == DAX_BF16>(r.y);
    f.v[2] = f2_from16<DT == DAX_BF16>(r.z);
    f.v[3] = f2_from16<DT == DAX_BF16>(r.w);
  }
  return f;
}
template <int DT>
__device__ __forceinline__ uint4 pack(const Pairs<DT>& f) {
  if constexpr (DT == DAX_F32) {
    float a, b, c, d;
    f2_unpack(f.v[0], a, b);
    f2_unpack(f.v[1], c, d);
    return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d));
  } else {
    return make_uint4(f2_to16_rn<DT == DAX_BF16>(f.v[0]), f2_to16_rn<DT == DAX_BF16>(f.v[1]), f2_to16_rn<DT == DAX_BF16>(f.v[2]),
                      f2_to16_rn<DT == DAX_BF16>(f.v[3]));
  }
}
// the channels of a piece of a per-channel fp32 vector
template <int DT>
__device__ __forceinline__ Pairs<DT> load_vector(const float* p) {
  Pairs<DT> f;
#pragma unroll
  for (int k = 0; k < Piece<DT>::value / 4; ++k) {
    const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(p + 4 * k);
    f.v[2 * k] = u.x;
    f.v[2 * k + 1] = u.y;
  }
  return f;
}
template <int DT>
__device__ __forceinline__ void store_vector(float* p, const Pairs<DT>& f) {
#pragma unroll
  for (int k = 0; k < Piece<DT>::value / 4; ++k) *reinterpret_cast<ulonglong2*>(p + 4 * k) = make_ulonglong2(f.v[2 * k], f.v[2 * k + 1]);
}
__device__ __forceinline__ float f2_sum(uint64_t p) {
  float a, b;
  f2_unpack(p, a, b);
  return a + b;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sums of N values over the CTA, the same numbers in every thread.  `slots` (one per warp the CTA may have, those of absent
// warps zero) may be written again after the next barrier: callers alternate between two sets, so one barrier per reduction
// is enough.
template <int N> struct alignas(N * 4) Sums { float v[N]; };
template <int N, int WARPS>
__device__ __forceinline__ void cta_sum(float (&v)[N], Sums<N>* slots) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = warp_sum(v[k]);
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) slots[threadIdx.x >> 5].v[k] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const Sums<N> s = slots[w];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += s.v[k];
  }
}

// The rotary factors of this thread's pairs: a head has 128 channels and blockDim.x pieces are a whole number of heads,
// so all pieces of a thread sit at the same channels of their heads and share the factors.
template <int DT> struct Rotary { float c[Piece<DT>::value / 2], s[Piece<DT>::value / 2]; };
template <int DT>
__device__ __forceinline__ void load_rotary(const NormArgs& p, int64_t row, Rotary<DT>& r) {
  constexpr int E = Piece<DT>::value;
  const int pair = (threadIdx.x * E % 128) / 2;
#pragma unroll
  for (int k = 0; k < E / 2; k += 2) {
    *reinterpret_cast<float2*>(&r.c[k]) = *reinterpret_cast<const float2*>(p.cos + row * 64 + pair + k);
    *reinterpret_cast<float2*>(&r.s[k]) = *reinterpret_cast<const float2*>(p.sin + row * 64 + pair + k);
  }
}

// Rotation of the piece's pairs by their angles (SIGN 1) or back (SIGN -1).
template <int DT, int SIGN>
__device__ __forceinline__ void rotate(Pairs<DT>& f, const Rotary<DT>& r) {
#pragma unroll
  for (int k = 0; k < Piece<DT>::value / 2; ++k) {
    float u, w;
    f2_unpack(f.v[k], u, w);
    const float s = SIGN > 0 ? r.s[k] : -r.s[k];
    f.v[k] = f2_pack(fmaf(u, r.c[k], -(w * s)), fmaf(w, r.c[k], u * s));
  }
}

// ---- launch shapes -----------------------------------------------------------------------------------------------------
// ELEMS elements of a row per thread (NV pieces), at most T threads, at least MINB CTAs per SM (which bounds the registers),
// R rows at a time, STAGES groups of rows in the ring.  Two rows at a time while the ring of two CTAs fits the SM: not for
// fp32 and not for the widest rows.
template <int DT, int ELEMS, bool BACKWARD> struct Shape {
  static constexpr int NV = ELEMS / Piece<DT>::value;
  static constexpr int T = ELEMS == 8 ? 128 : ELEMS == 16 ? 320 : 256;
  static constexpr int WARPS = T / 32;
  static constexpr int MINB = ELEMS == 8 ? 6 : 2;
  static constexpr int R = DT != DAX_F32 && ELEMS <= 16 ? 2 : 1;
  static constexpr int STAGES = BACKWARD ? 2 : 3;
};

// Pieces of a thread that lie behind the row's end, and rows behind the last one, are zeros in the ring: they add nothing to
// any sum, so only stores ask whether they exist.

// ---- forward ---------------------------------------------------------------------------------------------------------
template <int DT, int ELEMS, bool LN>
__global__ void __launch_bounds__(Shape<DT, ELEMS, false>::T, Shape<DT, ELEMS, false>::MINB) norm_forward_kernel(const NormArgs p) {
  using Sh = Shape<DT, ELEMS, false>;
  constexpr int E = Piece<DT>::value, NV = Sh::NV, R = Sh::R, STAGES = Sh::STAGES, N = LN ? 2 * R : R, W = Sh::WARPS;
  extern __shared__ uint4 ring[];  // [STAGES][R][NV][blockDim.x], then the coefficients
  __shared__ Sums<N> red[2][W], red_c[2][W];
  const int T = blockDim.x, tid = threadIdx.x, b = blockIdx.y, S = static_cast<int>(p.S);
  const int mine = (p.D / E - tid + T - 1) / T;  // pieces of this thread
  const uint8_t* x = p.x + b * p.x_sb + tid * 16;
  uint8_t* y = p.out + b * p.out_sb + tid * 16;
  uint4* slot = ring + tid;
  for (int k = tid; k < 2 * W * N; k += T) {
    (&red[0][0].v[0])[k] = 0.f;
    (&red_c[0][0].v[0])[k] = 0.f;
  }

  auto fetch = [&](int row0, int stage) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint8_t* src = x + (row0 + r) * p.x_ss;
#pragma unroll
      for (int i = 0; i < NV; ++i) cp_async16(&slot[((stage * R + r) * NV + i) * T], src + i * T * 16, row0 + r < S && i < mine);
    }
    cp_async_commit();
  };
  const int step = gridDim.x * R;
  int row0 = blockIdx.x * R;
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) fetch(row0 + k * step, k);
  // y = n mul + add per channel: (n w + c) (1 + scale) + shift, folded once per CTA.  In shared memory and not read from
  // global memory for every row (from L1 they cost a quarter more time); a thread reads what it wrote itself
  const bool coef = p.weight != nullptr || p.scale != nullptr;
  ulonglong2* mul_s = reinterpret_cast<ulonglong2*>(ring + STAGES * R * NV * T) + tid;
  ulonglong2* add_s = mul_s + NV * (E / 4) * T;
  if (coef) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i >= mine) continue;
      const int at = (tid + i * T) * E;
      Pairs<DT> mul, add;
#pragma unroll
      for (int k = 0; k < E / 2; ++k) {
        mul.v[k] = f2_splat(1.f);
        add.v[k] = f2_splat(0.f);
      }
      if (p.weight != nullptr) mul = load_vector<DT>(p.weight + at);
      if (LN && p.bias != nullptr) add = load_vector<DT>(p.bias + at);
      if (LN && p.scale != nullptr) {
        const int64_t row = static_cast<int64_t>(b) * p.D + at;
        const Pairs<DT> t = load_vector<DT>(p.scale + row), u = load_vector<DT>(p.shift + row);
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          mul.v[k] = f2_fma(mul.v[k], t.v[k], mul.v[k]);
          add.v[k] = f2_add(f2_fma(add.v[k], t.v[k], add.v[k]), u.v[k]);
        }
      }
#pragma unroll
      for (int q = 0; q < E / 4; ++q) {
        mul_s[(i * (E / 4) + q) * T] = make_ulonglong2(mul.v[2 * q], mul.v[2 * q + 1]);
        if (LN) add_s[(i * (E / 4) + q) * T] = make_ulonglong2(add.v[2 * q], add.v[2 * q + 1]);
      }
    }
  }
  __syncthreads();  // the sums' slots are zero
  const float inv_d = 1.f / static_cast<float>(p.D);
  int stage = 0, parity = 0;
  for (; row0 < S; row0 += step) {
    fetch(row0 + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
    Rotary<DT> rot[R];
    if (!LN && p.cos != nullptr) {
#pragma unroll
      for (int r = 0; r < R; ++r) load_rotary<DT>(p, min(row0 + r, S - 1), rot[r]);
    }
    cp_async_wait<STAGES - 1>();  // this thread's pieces of the rows have landed
    Pairs<DT> f[R][NV];
    float sum[N];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      uint64_t q2 = f2_splat(0.f), s2 = f2_splat(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        f[r][i] = unpack<DT>(slot[((stage * R + r) * NV + i) * T]);
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          q2 = f2_fma(f[r][i].v[k], f[r][i].v[k], q2);
          if (LN) s2 = f2_add(s2, f[r][i].v[k]);
        }
      }
      sum[r] = f2_sum(q2);
      if (LN) sum[R + (LN ? r : 0)] = f2_sum(s2);
    }
    cta_sum<N, W>(sum, red[parity]);
    float mean[R], rstd[R];
    bool centre[R], any = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = LN ? sum[R + (LN ? r : 0)] * inv_d : 0.f;
      const float var = fmaf(-mean[r], mean[r], sum[r] * inv_d);
      centre[r] = LN && !(var >= 4.f * mean[r] * mean[r]);
      any = any || centre[r];
      rstd[r] = rsqrtf(var + p.eps);
    }
    if (LN && any) {
      // E[x^2] - mean^2 loses digits where the mean is not small against the spread (every thread sees the same numbers, so
      // the branch is uniform): a second pass around the first estimate of the mean.  It takes the rounding of that
      // estimate out as well, so that a constant row normalises to zero.  A row that does not need it keeps its first numbers:
      // its bits do not depend on the row beside it.
#pragma unroll
      for (int r = 0; r < R; ++r) {
        uint64_t q2 = f2_splat(0.f), s2 = f2_splat(0.f);
        const uint64_t nm = f2_splat(-mean[r]);
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (i < mine) {
#pragma unroll
            for (int k = 0; k < E / 2; ++k) {
              const uint64_t d = f2_add(f[r][i].v[k], nm);
              q2 = f2_fma(d, d, q2);
              s2 = f2_add(s2, d);
            }
          }
        sum[r] = f2_sum(q2);
        sum[R + (LN ? r : 0)] = f2_sum(s2);
      }
      cta_sum<N, W>(sum, red_c[parity]);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (!centre[r]) continue;
        const float dm = sum[R + (LN ? r : 0)] * inv_d;
        mean[r] += dm;
        rstd[r] = rsqrtf(fmaxf(fmaf(-dm, dm, sum[r] * inv_d), 0.f) + p.eps);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (tid == r && row0 + r < S) {
        if (LN) p.mean[static_cast<int64_t>(b) * S + row0 + r] = mean[r];
        p.rstd[static_cast<int64_t>(b) * S + row0 + r] = rstd[r];
      }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Pairs<DT> mul, add;
      if (coef) {
#pragma unroll
        for (int q = 0; q < E / 4; ++q) {
          const ulonglong2 m = mul_s[(i * (E / 4) + q) * T];
          mul.v[2 * q] = m.x;
          mul.v[2 * q + 1] = m.y;
          if (LN) {
            const ulonglong2 c = add_s[(i * (E / 4) + q) * T];
            add.v[2 * q] = c.x;
            add.v[2 * q + 1] = c.y;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint64_t nm = f2_splat(-mean[r]), rs = f2_splat(rstd[r]);
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          f[r][i].v[k] = f2_mul(LN ? f2_add(f[r][i].v[k], nm) : f[r][i].v[k], rs);
          if (coef) f[r][i].v[k] = LN ? f2_fma(f[r][i].v[k], mul.v[k], add.v[k]) : f2_mul(f[r][i].v[k], mul.v[k]);
        }
        if (!LN && p.cos != nullptr) rotate<DT, 1>(f[r][i], rot[r]);
        if (row0 + r < S && i < mine) *reinterpret_cast<uint4*>(y + (row0 + r) * p.out_ss + i * T * 16) = pack<DT>(f[r][i]);
      }
    }
    stage = stage == STAGES - 1 ? 0 : stage + 1;
    parity ^= 1;
  }
  cp_async_wait<0>();  // the zeros behind the last row have arrived before the CTA gives back its memory
}

// ---- backward --------------------------------------------------------------------------------------------------------
// SUMS: column sums kept (0: none wanted; LayerNorm 2: A and N; RMSNorm 1: N).
template <int DT, int ELEMS, bool LN, int SUMS>
__global__ void __launch_bounds__(Shape<DT, ELEMS, true>::T, Shape<DT, ELEMS, true>::MINB) norm_backward_kernel(const NormArgs p) {
  using Sh = Shape<DT, ELEMS, true>;
  constexpr int E = Piece<DT>::value, NV = Sh::NV, R = Sh::R, STAGES = Sh::STAGES, N = LN ? 2 * R : R, W = Sh::WARPS;
  extern __shared__ uint4 ring[];  // [STAGES][R][2][NV][blockDim.x], then the coefficients
  __shared__ Sums<N> red[2][W];
  const int T = blockDim.x, tid = threadIdx.x, b = blockIdx.y, S = static_cast<int>(p.S);
  const int mine = (p.D / E - tid + T - 1) / T;
  const uint8_t* x = p.x + b * p.x_sb + tid * 16;
  const uint8_t* dy = p.dy + b * p.dy_sb + tid * 16;
  uint8_t* dx = p.out + b * p.out_sb + tid * 16;
  uint4* slot = ring + tid;
  const float* mean_b = LN ? p.mean + static_cast<int64_t>(b) * S : nullptr;
  const float* rstd_b = p.rstd + static_cast<int64_t>(b) * S;
  for (int k = tid; k < 2 * W * N; k += T) (&red[0][0].v[0])[k] = 0.f;

  auto fetch = [&](int row0, int stage) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint8_t *src = x + (row0 + r) * p.x_ss, *src_g = dy + (row0 + r) * p.dy_ss;
      uint4* at = slot + (stage * R + r) * 2 * NV * T;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const bool valid = row0 + r < S && i < mine;
        cp_async16(at + i * T, src + i * T * 16, valid);
        cp_async16(at + (NV + i) * T, src_g + i * T * 16, valid);
      }
    }
    cp_async_commit();
  };
  const int step = gridDim.x * R;
  int row0 = blockIdx.x * R;
#pragma unroll
  for (int k = 0; k < STAGES - 1; ++k) fetch(row0 + k * step, k);

  const bool coef = p.weight != nullptr || p.scale != nullptr;  // g = dy mul, mul = w (1 + scale)
  ulonglong2* mul_s = reinterpret_cast<ulonglong2*>(ring + STAGES * R * 2 * NV * T) + tid;
  if (coef) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (tid + i * T) * E;
      Pairs<DT> mul;
#pragma unroll
      for (int k = 0; k < E / 2; ++k) mul.v[k] = f2_splat(1.f);  // behind the row's end: times zero
      if (i < mine) {
        if (p.weight != nullptr) mul = load_vector<DT>(p.weight + at);
        if (LN && p.scale != nullptr) {
          const Pairs<DT> t = load_vector<DT>(p.scale + static_cast<int64_t>(b) * p.D + at);
#pragma unroll
          for (int k = 0; k < E / 2; ++k) mul.v[k] = f2_fma(mul.v[k], t.v[k], mul.v[k]);
        }
      }
#pragma unroll
      for (int q = 0; q < E / 4; ++q) mul_s[(i * (E / 4) + q) * T] = make_ulonglong2(mul.v[2 * q], mul.v[2 * q + 1]);
    }
  }
  __syncthreads();  // the sums' slots are zero
  Pairs<DT> sum_n[SUMS > 0 ? NV : 1], sum_a[SUMS > 1 ? NV : 1];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
      if (SUMS > 0) sum_n[SUMS > 0 ? i : 0].v[k] = f2_splat(0.f);
      if (SUMS > 1) sum_a[SUMS > 1 ? i : 0].v[k] = f2_splat(0.f);
    }

  // n and `raw` = dy (rotated back) of piece i, and g = raw times the coefficients
  auto piece = [&](const uint4* at, int i, uint64_t nm, uint64_t rs, const Rotary<DT>& rot, Pairs<DT>& n, Pairs<DT>& raw, Pairs<DT>& g) {
    n = unpack<DT>(at[i * T]);
    raw = unpack<DT>(at[(NV + i) * T]);
    if (!LN && p.cos != nullptr) rotate<DT, -1>(raw, rot);
#pragma unroll
    for (int k = 0; k < E / 2; ++k) n.v[k] = f2_mul(LN ? f2_add(n.v[k], nm) : n.v[k], rs);
    g = raw;
    if (coef) {
#pragma unroll
      for (int q = 0; q < E / 4; ++q) {
        const ulonglong2 m = mul_s[(i * (E / 4) + q) * T];
        g.v[2 * q] = f2_mul(g.v[2 * q], m.x);
        g.v[2 * q + 1] = f2_mul(g.v[2 * q + 1], m.y);
      }
    }
  };

  const float inv_d = 1.f / static_cast<float>(p.D);
  int stage = 0, parity = 0;
  // the statistics of the rows are read one group ahead
  float mean_next[R], rstd_next[R];
  auto statistics = [&](int row) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int at = min(row + r, S - 1);
      mean_next[r] = LN ? mean_b[at] : 0.f;
      rstd_next[r] = rstd_b[at];
    }
  };
  statistics(min(row0, S - 1));
  for (; row0 < S; row0 += step) {
    fetch(row0 + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
    uint64_t nm[R], rs[R];
    Rotary<DT> rot[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      nm[r] = f2_splat(-mean_next[r]);
      rs[r] = f2_splat(rstd_next[r]);
      if (!LN && p.cos != nullptr) load_rotary<DT>(p, min(row0 + r, S - 1), rot[r]);
    }
    statistics(min(row0 + step, S - 1));
    cp_async_wait<STAGES - 1>();
    float sum[N];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      uint64_t s_gn = f2_splat(0.f), s_g = f2_splat(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        Pairs<DT> n, raw, g;
        piece(slot + (stage * R + r) * 2 * NV * T, i, nm[r], rs[r], rot[r], n, raw, g);
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          if (SUMS > 0) sum_n[SUMS > 0 ? i : 0].v[k] = f2_fma(raw.v[k], n.v[k], sum_n[SUMS > 0 ? i : 0].v[k]);
          if (SUMS > 1) sum_a[SUMS > 1 ? i : 0].v[k] = f2_add(sum_a[SUMS > 1 ? i : 0].v[k], raw.v[k]);
          s_gn = f2_fma(g.v[k], n.v[k], s_gn);
          if (LN) s_g = f2_add(s_g, g.v[k]);
        }
      }
      sum[r] = f2_sum(s_gn);
      if (LN) sum[R + (LN ? r : 0)] = f2_sum(s_g);
    }
    cta_sum<N, W>(sum, red[parity]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint64_t neg_gn = f2_splat(-sum[r] * inv_d), neg_g = f2_splat(LN ? -sum[R + (LN ? r : 0)] * inv_d : 0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        Pairs<DT> n, raw, g;
        piece(slot + (stage * R + r) * 2 * NV * T, i, nm[r], rs[r], rot[r], n, raw, g);
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          const uint64_t t = f2_fma(n.v[k], neg_gn, g.v[k]);
          g.v[k] = f2_mul(LN ? f2_add(t, neg_g) : t, rs[r]);
        }
        if (row0 + r < S && i < mine) *reinterpret_cast<uint4*>(dx + (row0 + r) * p.out_ss + i * T * 16) = pack<DT>(g);
      }
    }
    stage = stage == STAGES - 1 ? 0 : stage + 1;
    parity ^= 1;
  }
  cp_async_wait<0>();  // the zeros behind the last row have arrived before the CTA gives back its memory
  if constexpr (SUMS > 0) {
    float* part = p.part + (static_cast<int64_t>(b) * gridDim.x + blockIdx.x) * SUMS * p.D + tid * E;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i >= mine) continue;
      store_vector<DT>(part + i * T * E, sum_n[SUMS > 0 ? i : 0]);
      if (SUMS > 1) store_vector<DT>(part + p.D + i * T * E, sum_a[SUMS > 1 ? i : 0]);
    }
  }
}

// ---- column sums over the CTAs ---------------------------------------------------------------------------------------
// A block owns 16 channels (64 bytes of a row of partial sums): 32 thread rows add every 32nd of them with eight loads in
// flight, then the 32 results are added in a tree: always in the same order.  Latency is what counts here: with 32
// channels and 32 thread rows in half as many blocks, the results added up by one row, a join of 888 x 2 x 1,536 took 10.6 us
// instead of 8.4.
struct JoinArgs {
  const float* part;  // [B, ctas, SUMS, D]
  const float* weight;
  const float* bias;
  const float* scale;
  float* dweight;
  float* dbias;
  float* dshift;
  float* dscale;
  int B, ctas, D;
};
template <int SUMS>
__global__ void __launch_bounds__(512, 2) norm_join_kernel(const JoinArgs p) {
  __shared__ float sm[SUMS][16][17], res[2][16];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = blockIdx.x * 16 + tx;
  const bool in = n < p.D;
  const int64_t stride = static_cast<int64_t>(SUMS) * p.D;
  float dw = 0.f, dc = 0.f;
  for (int b = 0; b < p.B; ++b) {
    float s[SUMS] = {};
    if (in) {
      const float* q = p.part + b * p.ctas * stride + n;
      for (int c = ty; c < p.ctas; c += 256) {  // eight rows' loads at a time
        float u[SUMS][8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int i = 0; i < SUMS; ++i) u[i][k] = c + 32 * k < p.ctas ? __ldcg(q + (c + 32 * k) * stride + i * p.D) : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int i = 0; i < SUMS; ++i) s[i] += u[i][k];
      }
    }
#pragma unroll
    for (int i = 0; i < SUMS; ++i) {
      s[i] += __shfl_xor_sync(0xffffffffu, s[i], 16);
      if (lane < 16) sm[i][warp][tx] = s[i];
    }
    __syncthreads();
    if (warp < 8 * SUMS) {  // half a warp adds the 16 warps' parts of one sum of one channel
      const int i = warp >> 3, c = 2 * (warp & 7) + (lane >> 4);
      float t = sm[i][tx][c];
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      if (tx == 0) res[i][c] = t;
    }
    __syncthreads();
    if (threadIdx.x < 16 && in) {
      const float s_n = res[0][tx], s_a = SUMS > 1 ? res[1][tx] : 0.f;
      const int64_t at = static_cast<int64_t>(b) * p.D + n;
      const float m = p.scale != nullptr ? 1.f + p.scale[at] : 1.f;
      if (p.dshift != nullptr) p.dshift[at] = s_a;
      if (p.dscale != nullptr) {
        const float w = p.weight != nullptr ? p.weight[n] : 1.f, c = p.bias != nullptr ? p.bias[n] : 0.f;
        p.dscale[at] = fmaf(w, s_n, c * s_a);
      }
      dw = fmaf(m, s_n, dw);
      dc = fmaf(m, s_a, dc);
    }
  }
  if (threadIdx.x < 16 && in) {
    if (p.dweight != nullptr) p.dweight[n] = dw;
    if (p.dbias != nullptr) p.dbias[n] = dc;
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------------
// Elements of a row per thread: few while the rows are narrow, so that there are threads; at most 320 threads.  Between
// 2,560 and 5,120 channels 16 and 32 both fit; which is faster goes by the registers that the pass needs beside the row
// (32,760 x 5,120 bf16, us, 16 / 32: LayerNorm forward 117 / 124, backward 205 / 193, RMSNorm 118 / 112 and 211 / 225;
// fp32 6,240 rows, LayerNorm: 52 / 54 and 89 / 104).  Between (2,688, 3,584, 4,096 and 4,608
// channels, tensors of 210 MB, us, smallest and largest time with 16 / with 32): bf16 LayerNorm forward 69-75 / 69-71, backward 134-142 /
// 112-129, RMSNorm forward 78-84 / 71-78, backward 138-150 / 132-149 (with 32 5 and 7 % faster at 3,584 and 4,096, slower at the
// others); fp32 LayerNorm 78-80 / 78-79 and 100-107 / 127-141, RMSNorm 77-81 / 70-76 (16 costs 6 to 12 % there) and 120-128 / 128-138.
inline int row_elems(int64_t D, int dtype, bool ln, bool backward) {
  return D <= 1024 ? 8 : (D <= (dtype != DAX_F32 && ln == backward ? 2560 : 5120) ? 16 : 32);
}
// CTAs that stay resident and stride over the rows, over all samples: at most what fits on the GPU at once and eight per SM
// (more adds nothing to the bytes in flight, but partial sums to join).
inline int64_t max_ctas(int64_t B, int64_t groups) { return std::min(groups, std::max<int64_t>(1, 8 * static_cast<int64_t>(sm_count()) / B)); }

template <auto kernel>
int launch_rows(const NormArgs& p, int64_t B, int threads, size_t smem, int rows, int64_t* ctas, cudaStream_t st) {
  // The CTAs that fit an SM, asked for again when the device or the launch shape changes.
  // (device + 1) << 48 | threads << 32 | shared memory << 8 | CTAs
  static std::atomic<uint64_t> last{0};
  int dev = 0;
  DAX_CUDA(cudaGetDevice(&dev));
  const uint64_t key = static_cast<uint64_t>(dev + 1) << 48 | static_cast<uint64_t>(threads) << 32 | static_cast<uint64_t>(smem) << 8;
  const uint64_t known = last.load(std::memory_order_relaxed);
  int per_sm = static_cast<int>(known & 0xff);
  if ((known & ~uint64_t{0xff}) != key) {
    // the same limit whatever the shape: calls of other threads may set it at the same time
    DAX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
    DAX_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem));
    last.store(key | static_cast<uint64_t>(per_sm), std::memory_order_relaxed);
  }
  *ctas = std::min(max_ctas(B, (p.S + rows - 1) / rows), std::max<int64_t>(1, static_cast<int64_t>(per_sm) * sm_count() / B));
  kernel<<<dim3(static_cast<unsigned>(*ctas), static_cast<unsigned>(B)), threads, smem, st>>>(p);
  DAX_CUDA(cudaGetLastError());
  return DAX_OK;
}

template <int DT, int ELEMS, bool LN>
int run_shape(const NormArgs& p, int64_t B, int64_t* ctas, int sums, bool backward, cudaStream_t st) {
  const int threads = ((p.D + ELEMS - 1) / ELEMS + 31) / 32 * 32;
  const size_t coef = p.weight != nullptr || p.scale != nullptr ? static_cast<size_t>(threads) * ELEMS * 4 : 0;  // one fp32 vector
  const size_t row = static_cast<size_t>(threads) * ELEMS * (DT == DAX_F32 ? 4 : 2);
  if (!backward) {
    using Sh = Shape<DT, ELEMS, false>;
    return launch_rows<norm_forward_kernel<DT, ELEMS, LN>>(p, B, threads, row * Sh::STAGES * Sh::R + (LN ? 2 : 1) * coef, Sh::R, ctas, st);
  }
  using Sh = Shape<DT, ELEMS, true>;
  const size_t smem = row * Sh::STAGES * Sh::R * 2 + coef;
  if (sums == 0) return launch_rows<norm_backward_kernel<DT, ELEMS, LN, 0>>(p, B, threads, smem, Sh::R, ctas, st);
  return launch_rows<norm_backward_kernel<DT, ELEMS, LN, LN ? 2 : 1>>(p, B, threads, smem, Sh::R, ctas, st);
}

template <bool LN>
int run_rows(const NormArgs& p, int dtype, int64_t B, int64_t* ctas, int sums, bool backward, cudaStream_t st) {
  const int elems = row_elems(p.D, dtype, LN, backward);
#define DAX_ROWS(DT, N) \
  if (dtype == DT && elems == N) return run_shape<DT, N, LN>(p, B, ctas, sums, backward, st)
  DAX_ROWS(DAX_BF16, 8); DAX_ROWS(DAX_BF16, 16); DAX_ROWS(DAX_BF16, 32);
  DAX_ROWS(DAX_F16, 8); DAX_ROWS(DAX_F16, 16); DAX_ROWS(DAX_F16, 32);
  DAX_ROWS(DAX_F32, 8); DAX_ROWS(DAX_F32, 16); DAX_ROWS(DAX_F32, 32);
#undef DAX_ROWS
  return fail(DAX_ERR_UNSUPPORTED, "norm: dtype %d is not BF16/F16/F32", dtype);
}

int check_rows(const char* what, int dtype, int64_t B, int64_t S, int64_t D) {
  DAX_REQUIRE(B >= 0 && S >= 0 && D > 0, DAX_ERR_INVALID, "%s: bad shape B=%lld S=%lld D=%lld", what, (long long)B, (long long)S, (long long)D);
  DAX_REQUIRE(dtype == DAX_BF16 || dtype == DAX_F16 || dtype == DAX_F32, DAX_ERR_UNSUPPORTED, "%s: dtype %d is not BF16/F16/F32", what, dtype);
  DAX_REQUIRE(D % 8 == 0 && D <= kMaxWidth, DAX_ERR_UNSUPPORTED, "%s: D=%lld must be a multiple of 8 and at most %lld", what,
              (long long)D, (long long)kMaxWidth);
  DAX_REQUIRE(B <= 65535, DAX_ERR_UNSUPPORTED, "%s: batch %lld exceeds 65535", what, (long long)B);
  DAX_REQUIRE(S < (1ll << 30), DAX_ERR_UNSUPPORTED, "%s: %lld rows per sample", what, (long long)S);
  return DAX_OK;
}
int check_tensor(const char* what, const char* name, const void* t, int64_t sb, int64_t ss, int dtype) {
  DAX_REQUIRE(t != nullptr, DAX_ERR_INVALID, "%s: %s is null", what, name);
  const int64_t e = dtype_bytes(dtype);
  DAX_REQUIRE(aligned16(t) && sb * e % 16 == 0 && ss * e % 16 == 0, DAX_ERR_ALIGN,
              "%s: %s must be 16-byte aligned, with sample and token strides of whole 16 bytes", what, name);
  return DAX_OK;
}
int check_vectors(const char* what, std::initializer_list<const void*> vs) {
  for (const void* v : vs) DAX_REQUIRE(aligned16(v), DAX_ERR_ALIGN, "%s: the per-channel vectors must be 16-byte aligned", what);
  return DAX_OK;
}
#define DAX_TRY(expr)              \
  do {                             \
    const int rc__ = (expr);       \
    if (rc__ != DAX_OK) return rc__; \
  } while (0)

template <bool LN>
int forward(NormArgs p, int dtype, int64_t B, int64_t D, cudaStream_t st) {
  if (B == 0 || p.S == 0) return DAX_OK;
  const int64_t e = dtype_bytes(dtype);
  p.D = static_cast<int>(D);
  p.x_sb *= e; p.x_ss *= e; p.out_sb *= e; p.out_ss *= e;
  int64_t ctas = 0;
  return run_rows<LN>(p, dtype, B, &ctas, 0, false, st);
}

template <bool LN>
int backward(const char* what, NormArgs p, JoinArgs j, int dtype, int64_t B, int64_t D, void* workspace, size_t bytes, cudaStream_t st) {
  const bool want = j.dweight != nullptr || j.dbias != nullptr || j.dshift != nullptr || j.dscale != nullptr;
  const int sums = want ? (LN ? 2 : 1) : 0;
  int64_t ctas = B > 0 ? max_ctas(B, p.S) : 0;
  if (want) {
    const size_t need = static_cast<size_t>(B) * ctas * sums * D * 4;
    DAX_REQUIRE(bytes >= need && (need == 0 || workspace != nullptr), DAX_ERR_INVALID,
                "%s: workspace of %zu bytes is smaller than the %zu required", what, bytes, need);
    DAX_REQUIRE(aligned16(workspace), DAX_ERR_ALIGN, "%s: workspace must be 16-byte aligned", what);
  }
  const int64_t e = dtype_bytes(dtype);
  p.D = static_cast<int>(D);
  p.x_sb *= e; p.x_ss *= e; p.dy_sb *= e; p.dy_ss *= e; p.out_sb *= e; p.out_ss *= e;
  p.part = static_cast<float*>(workspace);
  if (B > 0 && p.S > 0) DAX_TRY(run_rows<LN>(p, dtype, B, &ctas, sums, true, st));
  if (want) {
    j.part = p.part;
    j.B = static_cast<int>(B);
    j.ctas = static_cast<int>(ctas);
    j.D = p.D;
    norm_join_kernel<LN ? 2 : 1><<<static_cast<unsigned>((D + 15) / 16), 512, 0, st>>>(j);
    DAX_CUDA(cudaGetLastError());
  }
  return DAX_OK;
}

}  // namespace
}  // namespace dax

extern "C" {

size_t dax_norm_backward_workspace_bytes(int64_t B, int64_t S, int64_t D) {
  if (B <= 0 || S <= 0 || D <= 0 || D > dax::kMaxWidth) return 0;
  return static_cast<size_t>(B) * dax::max_ctas(B, S) * 2 * D * 4;
}

int dax_layernorm_modulate(const void* x, int dtype, int64_t B, int64_t S, int64_t D, int64_t x_sb, int64_t x_ss,
                           const float* ln_weight, const float* ln_bias, const float* shift, const float* scale, float eps,
                           void* y, int64_t y_sb, int64_t y_ss, float* mean, float* rstd, void* stream) {
  using namespace dax;
  const char* what = "layernorm_modulate";
  DAX_TRY(check_rows(what, dtype, B, S, D));
  if (B == 0 || S == 0) return DAX_OK;
  DAX_TRY(check_tensor(what, "x", x, x_sb, x_ss, dtype));
  DAX_TRY(check_tensor(what, "y", y, y_sb, y_ss, dtype));
  DAX_REQUIRE(mean != nullptr && rstd != nullptr, DAX_ERR_INVALID, "%s: mean and rstd are needed", what);
  DAX_REQUIRE((shift == nullptr) == (scale == nullptr), DAX_ERR_INVALID, "%s: shift and scale come together", what);
  DAX_REQUIRE(ln_bias == nullptr || ln_weight != nullptr, DAX_ERR_INVALID, "%s: bias needs weight", what);
  DAX_TRY(check_vectors(what, {ln_weight, ln_bias, shift, scale}));
  NormArgs p{};
  p.x = static_cast<const uint8_t*>(x); p.x_sb = x_sb; p.x_ss = x_ss;
  p.out = static_cast<uint8_t*>(y); p.out_sb = y_sb; p.out_ss = y_ss;
  p.weight = ln_weight; p.bias = ln_bias; p.shift = shift; p.scale = scale;
  p.mean = mean; p.rstd = rstd; p.S = S; p.eps = eps;
  return forward<true>(p, dtype, B, D, static_cast<cudaStream_t>(stream));
}

int dax_layernorm_modulate_backward(const void* dy, const void* x, int dtype, int64_t B, int64_t S, int64_t D, int64_t dy_sb,
                                    int64_t dy_ss, int64_t x_sb, int64_t x_ss, const float* mean, const float* rstd,
                                    const float* ln_weight, const float* ln_bias, const float* scale, void* dx, int64_t dx_sb,
                                    int64_t dx_ss, float* dweight, float* dbias, float* dshift, float* dscale, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  using namespace dax;
  const char* what = "layernorm_modulate_backward";
  DAX_TRY(check_rows(what, dtype, B, S, D));
  if (B > 0 && S > 0) {
    DAX_TRY(check_tensor(what, "x", x, x_sb, x_ss, dtype));
    DAX_TRY(check_tensor(what, "dy", dy, dy_sb, dy_ss, dtype));
    DAX_TRY(check_tensor(what, "dx", dx, dx_sb, dx_ss, dtype));
    DAX_REQUIRE(mean != nullptr && rstd != nullptr, DAX_ERR_INVALID, "%s: mean and rstd are needed", what);
  }
  DAX_REQUIRE(ln_bias == nullptr || ln_weight != nullptr, DAX_ERR_INVALID, "%s: bias needs weight", what);
  DAX_TRY(check_vectors(what, {ln_weight, ln_bias, scale}));
  NormArgs p{};
  p.x = static_cast<const uint8_t*>(x); p.x_sb = x_sb; p.x_ss = x_ss;
  p.dy = static_cast<const uint8_t*>(dy); p.dy_sb = dy_sb; p.dy_ss = dy_ss;
  p.out = static_cast<uint8_t*>(dx); p.out_sb = dx_sb; p.out_ss = dx_ss;
  p.weight = ln_weight; p.scale = scale;
  p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd); p.S = S;
  JoinArgs j{};
  j.weight = ln_weight; j.bias = ln_bias; j.scale = scale;
  j.dweight = dweight; j.dbias = dbias; j.dshift = dshift; j.dscale = dscale;
  return backward<true>(what, p, j, dtype, B, D, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int dax_rmsnorm_rope(const void* x, int dtype, int64_t B, int64_t S, int64_t D, int64_t x_sb, int64_t x_ss,
                     const float* norm_weight, const float* rope_cos, const float* rope_sin, float eps, void* y, int64_t y_sb,
                     int64_t y_ss, float* rstd, void* stream) {
  using namespace dax;
  const char* what = "rmsnorm_rope";
  DAX_TRY(check_rows(what, dtype, B, S, D));
  if (B == 0 || S == 0) return DAX_OK;
  DAX_TRY(check_tensor(what, "x", x, x_sb, x_ss, dtype));
  DAX_TRY(check_tensor(what, "y", y, y_sb, y_ss, dtype));
  DAX_REQUIRE(rstd != nullptr, DAX_ERR_INVALID, "%s: rstd is needed", what);
  DAX_REQUIRE((rope_cos == nullptr) == (rope_sin == nullptr), DAX_ERR_INVALID, "%s: rope_cos and rope_sin come together", what);
  DAX_REQUIRE(rope_cos == nullptr || D % 128 == 0, DAX_ERR_INVALID, "%s: a rotation needs D=%lld to be whole heads of 128", what, (long long)D);
  DAX_TRY(check_vectors(what, {norm_weight, rope_cos, rope_sin}));
  NormArgs p{};
  p.x = static_cast<const uint8_t*>(x); p.x_sb = x_sb; p.x_ss = x_ss;
  p.out = static_cast<uint8_t*>(y); p.out_sb = y_sb; p.out_ss = y_ss;
  p.weight = norm_weight; p.cos = rope_cos; p.sin = rope_sin;
  p.rstd = rstd; p.S = S; p.eps = eps;
  return forward<false>(p, dtype, B, D, static_cast<cudaStream_t>(stream));
}

int dax_rmsnorm_rope_backward(const void* dy, const void* x, int dtype, int64_t B, int64_t S, int64_t D, int64_t dy_sb,
                              int64_t dy_ss, int64_t x_sb, int64_t x_ss, const float* rstd, const float* norm_weight,
                              const float* rope_cos, const float* rope_sin, void* dx, int64_t dx_sb, int64_t dx_ss,
                              float* dweight, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace dax;
  const char* what = "rmsnorm_rope_backward";
  DAX_TRY(check_rows(what, dtype, B, S, D));
  if (B > 0 && S > 0) {
    DAX_TRY(check_tensor(what, "x", x, x_sb, x_ss, dtype));
    DAX_TRY(check_tensor(what, "dy", dy, dy_sb, dy_ss, dtype));
    DAX_TRY(check_tensor(what, "dx", dx, dx_sb, dx_ss, dtype));
    DAX_REQUIRE(rstd != nullptr, DAX_ERR_INVALID, "%s: rstd is needed", what);
  }
  DAX_REQUIRE((rope_cos == nullptr) == (rope_sin == nullptr), DAX_ERR_INVALID, "%s: rope_cos and rope_sin come together", what);
  DAX_REQUIRE(rope_cos == nullptr || D % 128 == 0, DAX_ERR_INVALID, "%s: a rotation needs D=%lld to be whole heads of 128", what, (long long)D);
  DAX_TRY(check_vectors(what, {norm_weight, rope_cos, rope_sin}));
  NormArgs p{};
  p.x = static_cast<const uint8_t*>(x); p.x_sb = x_sb; p.x_ss = x_ss;
  p.dy = static_cast<const uint8_t*>(dy); p.dy_sb = dy_sb; p.dy_ss = dy_ss;
  p.out = static_cast<uint8_t*>(dx); p.out_sb = dx_sb; p.out_ss = dx_ss;
  p.weight = norm_weight; p.cos = rope_cos; p.sin = rope_sin;
  p.rstd = const_cast<float*>(rstd); p.S = S;
  JoinArgs j{};
  j.weight = norm_weight;
  j.dweight = dweight;
  return backward<false>(what, p, j, dtype, B, D, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
