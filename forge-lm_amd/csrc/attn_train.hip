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
__global__ __launch_bounds__(256, sizeof(E) == 4 && HD == 128 && KS == 4 ? 1 : 2) void k_attn_forward(const AttnTrain a) {
  typedef AtMma<E, HD> M;
  typedef AtPlan<E, HD, KS, VEC> P;
  constexpr int N = HD < 64 ? HD : 64;  // dims joined at a time
  constexpr bool kAhead = sizeof(E) == 2 && HD <= 64;  // registers for the transposed operand before the exponentials
  constexpr int kJoin = KS == 4 ? 4 * 32 * (N + 3) * 4 : 0, kHalf = P::kBytes / 2;
  // KS == 1: [K, V] tiles, and the same for odd steps; KS == 4: the waves' K tiles, and their V tiles
  constexpr int kFirst = KS == 1 ? P::kBytes : kHalf > kJoin ? kHalf : kJoin;
  __shared__ __align__(1024) char smem[kFirst], odd[KS == 4 ? kHalf : P::kBufs == 2 ? P::kBytes : 16];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nqb = (a.T + P::kOwn - 1) / P::kOwn;
  const AtBlock at = at_block(blockIdx.x, a.B * a.H, a.ragged);
  const int b = at.g / a.H, h = at.g % a.H, kvh = h / (a.H / a.Hk);
  const int t0 = (nqb - 1 - at.blk) * P::kOwn, len = at_len(a, b);
  const int qw0 = t0 + (KS == 1 ? 32 * w : 0), q = qw0 + (lane & 31);
  const E* seq = static_cast<const E*>(a.qkv) + (size_t)b * a.T * a.qkv_cols;
  const E* kb = seq + (size_t)(a.H + kvh) * a.hd;
  const E* vb = kb + (size_t)a.Hk * a.hd;
  const float sl2 = a.scale * kLog2e;
  at_f32x16 o[HD / 32];
#pragma unroll
  for (int dt = 0; dt < HD / 32; dt++) at_zero(o[dt]);
  float m = -INFINITY, l = 0.f;  // running maximum of scale * log2(e) * s, and sum

  if (t0 < len) {
    const typename M::Own own = M::template own<VEC>(
        at_rows(seq + (size_t)qw0 * a.qkv_cols + (size_t)h * a.hd, min(32, len - qw0), a.qkv_cols, a.hd), lane & 31, lane);
    auto rows_of = [&](const E* base, int k0) {
      return at_rows(base + (size_t)k0 * a.qkv_cols, min(P::kRows, len - k0), a.qkv_cols, a.hd);
    };
    // the 32 N keys from k0 on, tile rows r0 ..; the calls come where the K tile has been read for the last
    // time, and before the V tile is read
    auto part = [&](auto nparts, int k0, const E* Ks, const E* Vs, int r0, auto&& k_read, auto&& v_wait) {
      constexpr int N = decltype(nparts)::value;
      at_f32x16 s[N];
      typename M::Cols vf[N];
#pragma unroll
      for (int i = 0; i < N; i++) {
        at_zero(s[i]);
        M::rows(s[i], M::load_rows(Ks, r0 + 32 * i, lane), own);
      }
      k_read();
      v_wait();
#pragma unroll
      for (int i = 0; i < N; i++)
        if (kAhead) vf[i] = M::load_cols(Vs, r0 + 32 * i, lane);
      if (N == 1 && k0 + 31 > qw0) {                // the part crosses the diagonal
        const int left = q - k0 - 4 * (lane >> 5);  // at_row0 of the last key that the query sees
#pragma unroll
        for (int r = 0; r < 16; r++)
          if (at_row0(r) > left) s[0][r] = -INFINITY;
      }
      float mt = -INFINITY;
#pragma unroll
      for (int i = 0; i < N; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) mt = fmaxf(mt, s[i][r]);
      mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
      const float mn = fmaxf(m, mt * sl2);
      const float mr = mn == -INFINITY ? 0.f : mn;  // a query that has seen no key yet
      if (__builtin_amdgcn_ballot_w64(mn > m)) {    // a maximum of the wave has grown
        const float corr = __builtin_amdgcn_exp2f(m - mr);
        l *= corr;
        m = mn;
#pragma unroll
        for (int dt = 0; dt < HD / 32; dt++)
#pragma unroll
          for (int r = 0; r < 16; r++) o[dt][r] *= corr;
      }
      float ls = 0.f;
#pragma unroll
      for (int i = 0; i < N; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          s[i][r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], sl2, -mr));
          ls += s[i][r];
        }
      l += ls;
#pragma unroll
      for (int i = 0; i < N; i++) {
        if (!kAhead) vf[i] = M::load_cols(Vs, r0 + 32 * i, lane);
        M::cols(o, vf[i], s[i], lane);
      }
    };
    if constexpr (KS == 1) {
      auto fetch = [&](int kt, char* buf) {
        E* t = reinterpret_cast<E*>(buf);
        at_load<E, HD, KS, VEC>(t, rows_of(kb, kt * P::kRows), w, lane);
        at_load<E, HD, KS, VEC>(t + P::kTile, rows_of(vb, kt * P::kRows), w, lane);
      };
      auto compute = [&](int kt, const char* buf) {
        const E* t = reinterpret_cast<const E*>(buf);
        const int k0 = kt * P::kRows;
        if (k0 + P::kRows - 1 <= qw0) {  // every query of this wave sees all of it
          part(at_int<P::kParts>, k0, t, t + P::kTile, 0, [] {}, [] {});
          return;
        }
#pragma unroll
        for (int n = 0; n < P::kParts; n++)
          if (k0 + 32 * n <= qw0 + 31)  // some query does
            part(at_int<1>, k0 + 32 * n, t, t + P::kTile, 32 * n, [] {}, [] {});
      };
      at_walk<P>((min(t0 + P::kOwn, len) - 1) / P::kRows + 1, smem, odd, fetch, compute);
    } else {
      E *Ks = reinterpret_cast<E*>(smem) + w * P::kTile, *Vs = reinterpret_cast<E*>(odd) + w * P::kTile;
      const int last = t0 / 32;
      if (w <= last) {
        at_load<E, HD, KS, VEC>(Ks, rows_of(kb, 32 * w), 0, lane);
        at_load<E, HD, KS, VEC>(Vs, rows_of(vb, 32 * w), 0, lane);
      }
      for (int p = w; p <= last; p += 4) {  // (past the last part nothing is in reach, and zeros arrive)
        at_wait<P::kLoads>();
        part(at_int<1>, 32 * p, Ks, Vs, 0,
             [&] {
               at_wait<-1>();
               at_load<E, HD, KS, VEC>(Ks, rows_of(kb, 32 * (p + 4)), 0, lane);
             },
             [&] { at_wait<P::kLoads>(); });
        at_wait<-1>();
        at_load<E, HD, KS, VEC>(Vs, rows_of(vb, 32 * (p + 4)), 0, lane);
      }
    }
    l += __shfl_xor(l, 32, 64);
  }

  E* out = static_cast<E*>(a.out) + ((size_t)b * a.T + t0) * a.out_cols + (size_t)h * a.hd;
  float* lse = a.lse + (size_t)at.g * a.T;
  if constexpr (KS == 1) {
    at_landed();  // the tiles' LDS is free
    if (qw0 >= a.T) return;
    const bool row = q < len;
    at_store<E, HD, VEC, P::kStaged>(out + (size_t)32 * w * a.out_cols, a.out_cols, o, row ? 1.f / l : 0.f, a.T - qw0, len - qw0, a.hd,
                         reinterpret_cast<E*>(smem) + w * 32 * HD, lane);
    if (lane < 32 && q < a.T) lse[q] = row ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
  } else {
    // join: each wave's sums at the block's maximum
    float* om = reinterpret_cast<float*>(smem);  // [4][32] maxima, [4][32] sums, [4][32][N + 1] outputs
    float* ol = om + 128;
    float* os = ol + 128;
    at_landed();
    if (lane < 32) om[w * 32 + lane] = m;
    __syncthreads();
    float mx = om[lane & 31];
#pragma unroll
    for (int i = 1; i < 4; i++) mx = fmaxf(mx, om[i * 32 + (lane & 31)]);
    const float f = __builtin_amdgcn_exp2f(m - (mx == -INFINITY ? 0.f : mx));
    if (lane < 32) ol[w * 32 + lane] = l * f;
#pragma unroll
    for (int d0 = 0; d0 < HD; d0 += N) {
      if (d0) __syncthreads();
#pragma unroll
      for (int dt = 0; dt < N / 32; dt++)
#pragma unroll
        for (int r = 0; r < 16; r++)
          os[(w * 32 + (lane & 31)) * (N + 1) + dt * 32 + at_row(lane, r)] = o[d0 / 32 + dt][r] * f;
      __syncthreads();
      for (int e = tid; e < 32 * N; e += 256) {
        const int i = e / N, d = e % N;
        if (t0 + i >= a.T) break;
        if (d0 + d >= a.hd) continue;
        const float sum = ol[i] + ol[32 + i] + ol[64 + i] + ol[96 + i];
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < 4; k++) v += os[(k * 32 + i) * (N + 1) + d];
        out[(size_t)i * a.out_cols + d0 + d] = (E)(t0 + i < len ? v / sum : 0.f);
      }
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
