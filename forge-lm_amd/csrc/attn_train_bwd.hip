// attn_train_bwd.hip -- the backward pass of attn_train.hip, which computes the probabilities again
// from the scores and the forward's lse (gfx950).
//
//   p_ij = exp(scale q_i . k_j - lse_i)   D_i = do_i . o_i        ds_ij = p_ij (do_i . v_j - D_i)
//   dv_j = sum_i p_ij do_i                dq_i = scale sum_j ds_ij k_j   dk_j = scale sum_i ds_ij q_i
// One kernel takes blocks of queries and walks the keys (dq, and D for the other), one takes blocks of
// keys and walks the queries of every head that shares them (dk, dv).  The scores and dP are computed in
// both, 14 hd operations a visible pair where 10 would do, so that every gradient is summed by one
// block in a fixed order: no atomics, the same bits on every run.
#include "attn_train.hpp"

#include <math.h>

namespace fh {

namespace {

// The sum over the four waves of acc^T (dims x the 32 own rows), times f, to rows row0 .. of dst;
// rows at or past len are zeros, rows at or past T are not written.
template <typename E, int HD>
__device__ __forceinline__ void join_store(float* os, const at_f32x16 (&acc)[HD / 32], float f, E* dst, int row0, int len,
                                           int T, int stride, int hd, int w, int lane, int tid) {
  __syncthreads();
#pragma unroll
  for (int dt = 0; dt < HD / 32; dt++)
#pragma unroll
    for (int r = 0; r < 16; r++) os[(w * 32 + (lane & 31)) * (HD + 1) + dt * 32 + at_row(lane, r)] = acc[dt][r];
  __syncthreads();
  for (int e = tid; e < 32 * HD; e += 256) {
    const int i = e / HD, d = e % HD;
    if (row0 + i >= T) break;
    if (d >= hd) continue;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++) v += os[(k * 32 + i) * (HD + 1) + d];
    dst[(size_t)(row0 + i) * stride + d] = (E)(row0 + i < len ? v * f : 0.f);
  }
}

// lse and D of the rows as the other kernel reads them, [head][32-row part][32 of lse * log2(e), 32 of
// D]; rows past the length have lse +infinity (their p is 0) and D 0, parts past it are not written.
__device__ __forceinline__ float* stat_part(const AttnTrain& a, size_t head, int row) {
  return a.stats + (head * ((a.T + 31) / 32) + row / 32) * 64;
}

template <typename E, int HD, int KS, bool VEC>
__global__ __launch_bounds__(256) void k_attn_backward_q(const AttnTrain a) {
  typedef AtMma<E, HD> M;
  typedef AtPlan<E, HD, KS, VEC> P;
  constexpr int kJoin = KS == 4 ? 4 * 32 * (HD + 1) * 4 : 0;
  __shared__ __align__(1024) char smem[P::kBytes > kJoin ? P::kBytes : kJoin], odd[P::kBufs == 2 ? P::kBytes : 16];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nqb = (a.T + P::kOwn - 1) / P::kOwn;
  const AtBlock at = at_block(blockIdx.x, a.B * a.H);
  const int b = at.g / a.H, h = at.g % a.H, kvh = h / (a.H / a.Hk);
  const int t0 = (nqb - 1 - at.blk) * P::kOwn, len = at_len(a, b);
  const int qw0 = t0 + (KS == 1 ? 32 * w : 0), q = qw0 + (lane & 31);
  const size_t row0 = (size_t)b * a.T;
  const E* seq = static_cast<const E*>(a.qkv) + row0 * a.qkv_cols;
  const E* kb = seq + (size_t)(a.H + kvh) * a.hd;
  const E* vb = kb + (size_t)a.Hk * a.hd;
  const float sl2 = a.scale * kLog2e;
  const int mine = KS == 4 ? w * 2 * P::kTile : 0;  // this wave's K and V tiles in a buffer

  at_f32x16 dq[HD / 32];
#pragma unroll
  for (int dt = 0; dt < HD / 32; dt++) at_zero(dq[dt]);

  if (t0 < len) {
    const int nkt = (min(t0 + P::kOwn, len) - 1) / P::kRows + 1;
    auto fetch = [&](int kt, char* buf) {
      const int k0 = kt * P::kRows + (KS == 4 ? 32 * w : 0), n = min(KS == 4 ? 32 : P::kRows, len - k0);
      at_load<E, HD, KS, VEC>(reinterpret_cast<E*>(buf) + mine, at_rows(kb + (size_t)k0 * a.qkv_cols, n, a.qkv_cols, a.hd),
                              at_rows(vb + (size_t)k0 * a.qkv_cols, n, a.qkv_cols, a.hd), w, lane);
    };
    const int n = min(32, len - qw0);
    const typename M::Own own = M::template own<VEC>(
        at_rows(seq + (size_t)qw0 * a.qkv_cols + (size_t)h * a.hd, n, a.qkv_cols, a.hd), lane & 31, lane);
    const size_t orow = (row0 + qw0) * a.out_cols + (size_t)h * a.hd;
    const typename M::Own dout =
        M::template own<VEC>(at_rows(static_cast<const E*>(a.dout) + orow, n, a.out_cols, a.hd), lane & 31, lane);
    float D = M::dot(dout, M::template own<VEC>(at_rows(static_cast<const E*>(a.out) + orow, n, a.out_cols, a.hd),
                                                lane & 31, lane));
    D += __shfl_xor(D, 32, 64);
    const float lse2 = q < len ? a.lse[(size_t)at.g * a.T + q] * kLog2e : INFINITY;
    if ((KS == 1 || w == 0) && qw0 < len) stat_part(a, at.g, qw0)[lane] = lane < 32 ? lse2 : D;
    auto compute = [&](int kt, const char* buf) {
      const E *Ks = reinterpret_cast<const E*>(buf) + mine, *Vs = Ks + P::kTile;
#pragma unroll
      for (int i = 0; i < P::kParts; i++) {
        const int k0 = kt * P::kRows + 32 * (KS == 1 ? i : w);
        if (k0 > qw0 + 31) continue;
        at_f32x16 s, dp;
        at_zero(s);
        at_zero(dp);
        M::rows(s, Ks, 32 * i, own, lane);
        M::rows(dp, Vs, 32 * i, dout, lane);
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sl2, -lse2)) * (dp[r] - D);
        if (k0 + 31 > qw0) {  // the part crosses the diagonal
#pragma unroll
          for (int r = 0; r < 16; r++)
            if (k0 + at_row(lane, r) > q) s[r] = 0.f;
        }
        M::cols(dq, Ks, 32 * i, s, lane);
      }
    };
    at_walk<P, KS>(nkt, smem, odd, fetch, compute);
  }
  E* dst = static_cast<E*>(a.dqkv) + row0 * a.qkv_cols + (size_t)h * a.hd;
  if constexpr (KS == 1) {
    if (q >= a.T) return;
    if (q >= len)
#pragma unroll
      for (int dt = 0; dt < HD / 32; dt++) at_zero(dq[dt]);
    at_store<E, HD, VEC>(dst + (size_t)q * a.qkv_cols, dq, a.scale, a.hd, lane);
  } else {
    join_store<E, HD>(reinterpret_cast<float*>(smem), dq, a.scale, dst, t0, len, a.T, a.qkv_cols, a.hd, w, lane, tid);
  }
}

template <typename E, int HD, int KS, bool VEC>
__global__ __launch_bounds__(256) void k_attn_backward_kv(const AttnTrain a) {
  typedef AtMma<E, HD> M;
  typedef AtPlan<E, HD, KS, VEC> P;
  constexpr int kJoin = KS == 4 ? 4 * 32 * (HD + 1) * 4 : 0;
  __shared__ __align__(1024) char smem[P::kBytes > kJoin ? P::kBytes : kJoin], odd[P::kBufs == 2 ? P::kBytes : 16];
  __shared__ __align__(1024) float stat[P::kRows / 32][64], stat_odd[P::kRows / 32][64];  // of a buffer's parts

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const AtBlock at = at_block(blockIdx.x, a.B * a.Hk);
  const int b = at.g / a.Hk, kvh = at.g % a.Hk, group = a.H / a.Hk;
  const int k0 = at.blk * P::kOwn, len = at_len(a, b);
  const int kw0 = k0 + (KS == 1 ? 32 * w : 0), key = kw0 + (lane & 31);
  const size_t row0 = (size_t)b * a.T;
  const E* seq = static_cast<const E*>(a.qkv) + row0 * a.qkv_cols;
  const float sl2 = a.scale * kLog2e;
  const int mine = KS == 4 ? w * 2 * P::kTile : 0;  // this wave's Q and dO tiles in a buffer

  at_f32x16 dk[HD / 32], dv[HD / 32];
#pragma unroll
  for (int dt = 0; dt < HD / 32; dt++) {
    at_zero(dk[dt]);
    at_zero(dv[dt]);
  }
  if (k0 < len) {
    const int nqt = (len - k0 + P::kRows - 1) / P::kRows, nt = nqt * group;  // a head's tiles, all tiles
    int fg = 0, fq = k0;  // head of the group and first row of the tile to be fetched next
    auto fetch = [&](int, char* buf) {
      float(*sp)[64] = buf == smem ? stat : stat_odd;
      const int h = kvh * group + fg, q0 = fq + (KS == 4 ? 32 * w : 0), n = min(KS == 4 ? 32 : P::kRows, len - q0);
      const E* qb = seq + (size_t)q0 * a.qkv_cols + (size_t)h * a.hd;
      const E* ob = static_cast<const E*>(a.dout) + (row0 + q0) * a.out_cols + (size_t)h * a.hd;
      at_load<E, HD, KS, VEC>(reinterpret_cast<E*>(buf) + mine, at_rows(qb, n, a.qkv_cols, a.hd),
                              at_rows(ob, n, a.out_cols, a.hd), w, lane);
      // 32-row parts of the statistics: a wave's own, or one for each of the first waves
      const int part = fq + 32 * w;
      if ((KS == 4 || w < P::kRows / 32) && part < len) {
        if constexpr (VEC)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(
              at_rows(stat_part(a, (size_t)b * a.H + h, part), 1, 64, 64).rsrc,
              (__attribute__((address_space(3))) void*)&sp[w][0], 4, lane * 4, 0, 0, 0);
        else
          sp[w][lane] = stat_part(a, (size_t)b * a.H + h, part)[lane];
      }
      fq += P::kRows;
      if (fq >= len) {
        fq = k0;
        fg++;
      }
    };
    const int n = min(32, len - kw0);
    const E* kb = seq + (size_t)kw0 * a.qkv_cols + (size_t)(a.H + kvh) * a.hd;
    const typename M::Own ko = M::template own<VEC>(at_rows(kb, n, a.qkv_cols, a.hd), lane & 31, lane);
    const typename M::Own vo =
        M::template own<VEC>(at_rows(kb + (size_t)a.Hk * a.hd, n, a.qkv_cols, a.hd), lane & 31, lane);
    int q0 = k0;
    auto compute = [&](int, const char* buf) {
      const float(*sp)[64] = buf == smem ? stat : stat_odd;
      const E *Qs = reinterpret_cast<const E*>(buf) + mine, *Os = Qs + P::kTile;
#pragma unroll
      for (int i = 0; i < P::kParts; i++) {
        const int part = KS == 1 ? i : w, r0 = q0 + 32 * part;  // the part's first query
        if (r0 + 31 < kw0 || r0 >= len) continue;  // every query of it is before these keys, or past the length
        at_f32x16 s, dp;
        at_zero(s);
        at_zero(dp);
        M::rows(s, Qs, 32 * i, ko, lane);
        M::rows(dp, Os, 32 * i, vo, lane);
        const float* st = &sp[part][4 * (lane >> 5)];
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const float4 ls = *reinterpret_cast<const float4*>(st + 8 * c), ds = *reinterpret_cast<const float4*>(st + 32 + 8 * c);
          const float l4[4] = {ls.x, ls.y, ls.z, ls.w}, d4[4] = {ds.x, ds.y, ds.z, ds.w};
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int r = 4 * c + e;
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sl2, -l4[e]));
            dp[r] = s[r] * (dp[r] - d4[e]);
          }
        }
        if (r0 < kw0 + 31) {  // the part crosses the diagonal
#pragma unroll
          for (int r = 0; r < 16; r++)
            if (key > r0 + at_row(lane, r)) s[r] = dp[r] = 0.f;
        }
        M::cols(dv, Os, 32 * i, s, lane);
        M::cols(dk, Qs, 32 * i, dp, lane);
      }
      q0 += P::kRows;
      if (q0 >= len) q0 = k0;
    };
    at_walk<P, KS>(nt, smem, odd, fetch, compute);
  }
  E* dst = static_cast<E*>(a.dqkv) + row0 * a.qkv_cols + (size_t)(a.H + kvh) * a.hd;
  E* dstv = dst + (size_t)a.Hk * a.hd;
  if constexpr (KS == 1) {
    if (key >= a.T) return;
    if (key >= len)
#pragma unroll
      for (int dt = 0; dt < HD / 32; dt++) {
        at_zero(dk[dt]);
        at_zero(dv[dt]);
      }
    at_store<E, HD, VEC>(dst + (size_t)key * a.qkv_cols, dk, a.scale, a.hd, lane);
    at_store<E, HD, VEC>(dstv + (size_t)key * a.qkv_cols, dv, 1.f, a.hd, lane);
  } else {
    float* os = reinterpret_cast<float*>(smem);
    join_store<E, HD>(os, dk, a.scale, dst, k0, len, a.T, a.qkv_cols, a.hd, w, lane, tid);
    join_store<E, HD>(os, dv, 1.f, dstv, k0, len, a.T, a.qkv_cols, a.hd, w, lane, tid);
  }
}

template <typename E, int HD>
void backward_hd(hipStream_t st, const AttnTrain& a, bool vec, int cus) {
  const size_t wide = (size_t)((a.T + 127) / 128), narrow = (size_t)((a.T + 31) / 32);
  const size_t gq = (size_t)a.B * a.H, gk = (size_t)a.B * a.Hk;
  if (!vec) {
    hipLaunchKernelGGL((k_attn_backward_q<E, HD, 1, false>), dim3((unsigned)(wide * gq)), dim3(256), 0, st, a);
    hipLaunchKernelGGL((k_attn_backward_kv<E, HD, 1, false>), dim3((unsigned)(wide * gk)), dim3(256), 0, st, a);
    return;
  }
  if (wide * gq < (size_t)cus)
    hipLaunchKernelGGL((k_attn_backward_q<E, HD, 4, true>), dim3((unsigned)(narrow * gq)), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((k_attn_backward_q<E, HD, 1, true>), dim3((unsigned)(wide * gq)), dim3(256), 0, st, a);
  if (wide * gk < (size_t)cus)
    hipLaunchKernelGGL((k_attn_backward_kv<E, HD, 4, true>), dim3((unsigned)(narrow * gk)), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((k_attn_backward_kv<E, HD, 1, true>), dim3((unsigned)(wide * gk)), dim3(256), 0, st, a);
}

template <typename E>
void backward(hipStream_t st, const AttnTrain& a, bool vec, int cus) {
  if (a.hd <= 32)
    backward_hd<E, 32>(st, a, vec, cus);
  else if (a.hd <= 64)
    backward_hd<E, 64>(st, a, vec, cus);
  else
    backward_hd<E, 128>(st, a, vec, cus);
}

}  // namespace

hipError_t launch_attn_backward(hipStream_t st, const AttnTrain& a, bool bf16, int cus) {
  if (!attn_train_fits(a) || !a.qkv || !a.out || !a.lse || !a.dout || !a.dqkv || !a.stats) return hipErrorInvalidValue;
  const bool vec = attn_train_vec(a, bf16 ? 2 : 4);
  if (bf16)
    backward<__bf16>(st, a, vec, cus);
  else
    backward<float>(st, a, vec, cus);
  return hipGetLastError();
}

}  // namespace fh
