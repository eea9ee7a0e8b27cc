// attn_train.hip -- causal attention of packed q, k, v rows, forward (gfx950).
//
// Per (sequence, head), for a query i of the sequence's rows: s_ij = scale q_i . k_j for keys j <= i,
// o_i = sum_j exp(s_ij - lse_i) v_j with lse_i = log sum_j exp(s_ij).  One pass over the keys with a
// running maximum and sum; no score leaves the registers, and lse is all that the backward needs to
// compute the probabilities again.  Work: 4 hd operations a visible pair, q, k, v read and o written.
#include "attn_train.hpp"

#include <math.h>

namespace fh {

namespace {

template <typename E, int HD, int KS, bool VEC>
__global__ __launch_bounds__(256) void k_attn_forward(const AttnTrain a) {
  typedef AtMma<E, HD> M;
  typedef AtPlan<E, HD, KS, VEC> P;
  constexpr int kJoin = KS == 4 ? 4 * 32 * (HD + 3) * 4 : 0;
  __shared__ __align__(1024) char smem[P::kBytes > kJoin ? P::kBytes : kJoin], odd[P::kBufs == 2 ? P::kBytes : 16];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nqb = (a.T + P::kOwn - 1) / P::kOwn;
  const AtBlock at = at_block(blockIdx.x, a.B * a.H);
  const int b = at.g / a.H, h = at.g % a.H, kvh = h / (a.H / a.Hk);
  const int t0 = (nqb - 1 - at.blk) * P::kOwn, len = at_len(a, b);
  const int qw0 = t0 + (KS == 1 ? 32 * w : 0), q = qw0 + (lane & 31);
  const E* seq = static_cast<const E*>(a.qkv) + (size_t)b * a.T * a.qkv_cols;
  const E* kb = seq + (size_t)(a.H + kvh) * a.hd;
  const E* vb = kb + (size_t)a.Hk * a.hd;
  const float sl2 = a.scale * kLog2e;
  const int mine = KS == 4 ? w * 2 * P::kTile : 0;  // this wave's K and V tiles in a buffer

  at_f32x16 o[HD / 32];
#pragma unroll
  for (int dt = 0; dt < HD / 32; dt++) at_zero(o[dt]);
  float m = -INFINITY, l = 0.f;  // running maximum of scale * log2(e) * s, and sum

  if (t0 < len) {
    const typename M::Own own = M::template own<VEC>(
        at_rows(seq + (size_t)qw0 * a.qkv_cols + (size_t)h * a.hd, min(32, len - qw0), a.qkv_cols, a.hd), lane & 31, lane);
    const int nkt = (min(t0 + P::kOwn, len) - 1) / P::kRows + 1;
    auto fetch = [&](int kt, char* buf) {
      const int k0 = kt * P::kRows + (KS == 4 ? 32 * w : 0), n = min(KS == 4 ? 32 : P::kRows, len - k0);
      at_load<E, HD, KS, VEC>(reinterpret_cast<E*>(buf) + mine, at_rows(kb + (size_t)k0 * a.qkv_cols, n, a.qkv_cols, a.hd),
                              at_rows(vb + (size_t)k0 * a.qkv_cols, n, a.qkv_cols, a.hd), w, lane);
    };
    auto compute = [&](int kt, const char* buf) {
      const E *Ks = reinterpret_cast<const E*>(buf) + mine, *Vs = Ks + P::kTile;
#pragma unroll
      for (int n = 0; n < P::kParts; n++) {
        const int k0 = kt * P::kRows + 32 * (KS == 1 ? n : w);  // the part's first key
        if (k0 > qw0 + 31) continue;                            // no query of this wave sees it
        at_f32x16 s;
        at_zero(s);
        M::rows(s, Ks, 32 * n, own, lane);
        float mt = -INFINITY;
        if (k0 + 31 > qw0) {  // the part crosses the diagonal
#pragma unroll
          for (int r = 0; r < 16; r++)
            if (k0 + at_row(lane, r) > q) s[r] = -INFINITY;
        }
#pragma unroll
        for (int r = 0; r < 16; r++) {
          s[r] *= sl2;
          mt = fmaxf(mt, s[r]);
        }
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
        const float mn = fmaxf(m, mt);
        const float mr = mn == -INFINITY ? 0.f : mn;  // a query that has seen no key yet
        const float corr = __builtin_amdgcn_exp2f(m - mr);
        float ls = 0.f;
#pragma unroll
        for (int r = 0; r < 16; r++) {
          s[r] = __builtin_amdgcn_exp2f(s[r] - mr);
          ls += s[r];
        }
        l = l * corr + ls;
        m = mn;
#pragma unroll
        for (int dt = 0; dt < HD / 32; dt++)
#pragma unroll
          for (int r = 0; r < 16; r++) o[dt][r] *= corr;
        M::cols(o, Vs, 32 * n, s, lane);
      }
    };
    at_walk<P, KS>(nkt, smem, odd, fetch, compute);
    l += __shfl_xor(l, 32, 64);
  }

  E* out = static_cast<E*>(a.out) + ((size_t)b * a.T + q) * a.out_cols + (size_t)h * a.hd;
  float* lse = a.lse + (size_t)at.g * a.T;
  if constexpr (KS == 1) {
    if (q >= a.T) return;
    const bool row = q < len;
    if (!row)
#pragma unroll
      for (int dt = 0; dt < HD / 32; dt++) at_zero(o[dt]);
    at_store<E, HD, VEC>(out, o, row ? 1.f / l : 0.f, a.hd, lane);
    if (lane < 32) lse[q] = row ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
  } else {
    // join: each wave's sums at the block's maximum
    float* om = reinterpret_cast<float*>(smem);  // [4][32] maxima, [4][32] sums, [4][32][HD + 1] outputs
    float* ol = om + 128;
    float* os = ol + 128;
    __syncthreads();
    if (lane < 32) om[w * 32 + lane] = m;
    __syncthreads();
    float mx = om[lane & 31];
#pragma unroll
    for (int i = 1; i < 4; i++) mx = fmaxf(mx, om[i * 32 + (lane & 31)]);
    const float f = __builtin_amdgcn_exp2f(m - (mx == -INFINITY ? 0.f : mx));
    if (lane < 32) ol[w * 32 + lane] = l * f;
#pragma unroll
    for (int dt = 0; dt < HD / 32; dt++)
#pragma unroll
      for (int r = 0; r < 16; r++) os[(w * 32 + (lane & 31)) * (HD + 1) + dt * 32 + at_row(lane, r)] = o[dt][r] * f;
    __syncthreads();
    E* o0 = static_cast<E*>(a.out) + ((size_t)b * a.T + t0) * a.out_cols + (size_t)h * a.hd;
    for (int e = tid; e < 32 * HD; e += 256) {
      const int i = e / HD, d = e % HD;
      if (t0 + i >= a.T) break;
      if (d >= a.hd) continue;
      const float sum = ol[i] + ol[32 + i] + ol[64 + i] + ol[96 + i];
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < 4; k++) v += os[(k * 32 + i) * (HD + 1) + d];
      o0[(size_t)i * a.out_cols + d] = (E)(t0 + i < len ? v / sum : 0.f);
    }
    if (tid < 32 && t0 + tid < a.T) {
      const float sum = ol[tid] + ol[32 + tid] + ol[64 + tid] + ol[96 + tid];
      lse[t0 + tid] = t0 + tid < len ? (mx + __builtin_amdgcn_logf(sum)) * kLn2 : -INFINITY;
    }
  }
}

template <typename E, int HD>
void forward_hd(hipStream_t st, const AttnTrain& a, bool vec, int cus) {
  const size_t wide = (size_t)((a.T + 127) / 128) * a.B * a.H;
  const bool split = wide < (size_t)cus;
  const dim3 grid((unsigned)(split ? (size_t)((a.T + 31) / 32) * a.B * a.H : wide));
  if (!vec)
    hipLaunchKernelGGL((k_attn_forward<E, HD, 1, false>), dim3((unsigned)wide), dim3(256), 0, st, a);
  else if (split)
    hipLaunchKernelGGL((k_attn_forward<E, HD, 4, true>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((k_attn_forward<E, HD, 1, true>), grid, dim3(256), 0, st, a);
}

template <typename E>
void forward(hipStream_t st, const AttnTrain& a, bool vec, int cus) {
  if (a.hd <= 32)
    forward_hd<E, 32>(st, a, vec, cus);
  else if (a.hd <= 64)
    forward_hd<E, 64>(st, a, vec, cus);
  else
    forward_hd<E, 128>(st, a, vec, cus);
}

}  // namespace

bool attn_train_fits(const AttnTrain& a) {
  return a.B > 0 && a.T > 0 && a.Hk > 0 && a.H > 0 && a.H % a.Hk == 0 && a.hd > 0 && a.hd <= kAttnTrainHead &&
         a.T <= 1 << 24 && a.qkv_cols <= 1 << 20 && a.out_cols <= 1 << 20 && (size_t)a.B * a.H * ((a.T + 31) / 32) < 1u << 24;
}

hipError_t launch_attn_forward(hipStream_t st, const AttnTrain& a, bool bf16, int cus) {
  if (!attn_train_fits(a) || !a.qkv || !a.out || !a.lse) return hipErrorInvalidValue;
  const int es = bf16 ? 2 : 4;
  const bool vec = attn_train_vec(a, es);
  if (bf16)
    forward<__bf16>(st, a, vec, cus);
  else
    forward<float>(st, a, vec, cus);
  return hipGetLastError();
}

}  // namespace fh
