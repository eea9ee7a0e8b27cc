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
// rows at or past len are zeros, rows at or past T are not written.  os: kJoinFloats<HD>.
template <int HD>
constexpr int kJoinFloats = 4 * 32 * ((HD < 64 ? HD : 64) + 1);  // 64 dims at a time
template <typename E, int HD>
__device__ __forceinline__ void join_store(float* os, const at_f32x16 (&acc)[HD / 32], float f, E* dst, int row0, int len,
                                           int T, int stride, int hd, int w, int lane, int tid) {
  constexpr int N = HD < 64 ? HD : 64;
#pragma unroll
  for (int d0 = 0; d0 < HD; d0 += N) {
    at_landed();
#pragma unroll
    for (int dt = 0; dt < N / 32; dt++)
#pragma unroll
      for (int r = 0; r < 16; r++)
        os[(w * 32 + (lane & 31)) * (N + 1) + dt * 32 + at_row(lane, r)] = acc[d0 / 32 + dt][r];
    __syncthreads();
    for (int e = tid; e < 32 * N; e += 256) {
      const int i = e / N, d = e % N;
      if (row0 + i >= T) break;
      if (d0 + d >= hd) continue;
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < 4; k++) v += os[(k * 32 + i) * (N + 1) + d];
      dst[(size_t)(row0 + i) * stride + d0 + d] = (E)(row0 + i < len ? v * f : 0.f);
    }
  }
}

// lse and D of the rows as the other kernel reads them, [head][32-row part][32 of lse, 32 of D], both
// negated; lse times log2(e) (fp32: the exponent's addend) or by scale (bf16: where the product with k
// starts, which costs p some |lse| 2^-24 and saves an operation a score).  Rows past the length have lse
// +infinity (their p is 0) and D 0, parts past it are not written.
__device__ __forceinline__ float* stat_part(const AttnTrain& a, size_t head, int row) {
  return a.stats + (head * ((a.T + 31) / 32) + row / 32) * 64;
}

template <typename E, int HD, int KS, bool VEC>
__global__ __launch_bounds__(256, sizeof(E) == 4 && HD == 128 ? 1 : 2) void k_attn_backward_q(const AttnTrain a) {
  typedef AtMma<E, HD> M;
  typedef AtPlan<E, HD, KS, VEC> P;
  constexpr bool kAhead = sizeof(E) == 2 && HD <= 64;  // registers for the transposed operand before the exponentials
  constexpr int kJoin = KS == 4 ? kJoinFloats<HD> * 4 : 0, kHalf = P::kBytes / 2;
  // KS == 1: [K, V] tiles, and the same for odd steps; KS == 4: the waves' K tiles, and their V tiles
  constexpr int kFirst = KS == 1 ? P::kBytes : kHalf > kJoin ? kHalf : kJoin;
  __shared__ __align__(1024) char smem[kFirst], odd[KS == 4 ? kHalf : P::kBufs == 2 ? P::kBytes : 16];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nqb = (a.T + P::kOwn - 1) / P::kOwn;
  const AtBlock at = at_block(blockIdx.x, a.B * a.H, a.ragged);
  const int b = at.g / a.H, h = at.g % a.H, kvh = h / (a.H / a.Hk);
  const int t0 = (nqb - 1 - at.blk) * P::kOwn, len = at_len(a, b);
  const int qw0 = t0 + (KS == 1 ? 32 * w : 0), q = qw0 + (lane & 31);
  const size_t row0 = (size_t)b * a.T;
  const E* seq = static_cast<const E*>(a.qkv) + row0 * a.qkv_cols;
  const E* kb = seq + (size_t)(a.H + kvh) * a.hd;
  const E* vb = kb + (size_t)a.Hk * a.hd;
  const float sl2 = a.scale * kLog2e;

  at_f32x16 dq[HD / 32];
#pragma unroll
  for (int dt = 0; dt < HD / 32; dt++) at_zero(dq[dt]);

  if (t0 < len) {
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
    if ((KS == 1 || w == 0) && qw0 < len)
      stat_part(a, at.g, qw0)[lane] = lane >= 32 ? -D : sizeof(E) == 4 ? -lse2 : -lse2 / sl2;
    auto rows_of = [&](const E* base, int k0) {
      return at_rows(base + (size_t)k0 * a.qkv_cols, min(P::kRows, len - k0), a.qkv_cols, a.hd);
    };
    // the 32 keys from k0 on, tile rows r0 ..; the calls come where the V tile has been read for the last
    // time, and before the K tile is read
    auto part = [&](int k0, const E* Ks, const E* Vs, int r0, auto&& v_read, auto&& k_wait) {
      at_f32x16 s, dp;
      typename M::Cols kc;
      at_zero(dp);
      M::rows(dp, M::load_rows(Vs, r0, lane), dout);
      v_read();
      k_wait();
      at_zero(s);
      M::rows(s, M::load_rows(Ks, r0, lane), own);
      if (kAhead) kc = M::load_cols(Ks, r0, lane);
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sl2, -lse2)) * (dp[r] - D);
      if (k0 + 31 > qw0) {                          // the part crosses the diagonal
        const int left = q - k0 - 4 * (lane >> 5);  // at_row0 of the last key that the query sees
#pragma unroll
        for (int r = 0; r < 16; r++)
          if (at_row0(r) > left) s[r] = 0.f;
      }
      if (!kAhead) kc = M::load_cols(Ks, r0, lane);
      M::cols(dq, kc, s, lane);
    };
    if constexpr (KS == 1) {
      auto fetch = [&](int kt, char* buf) {
        E* t = reinterpret_cast<E*>(buf);
        at_load<E, HD, KS, VEC>(t, rows_of(kb, kt * P::kRows), w, lane);
        at_load<E, HD, KS, VEC>(t + P::kTile, rows_of(vb, kt * P::kRows), w, lane);
      };
      auto compute = [&](int kt, const char* buf) {
        const E* t = reinterpret_cast<const E*>(buf);
#pragma unroll
        for (int i = 0; i < P::kParts; i++) {
          const int k0 = kt * P::kRows + 32 * i;
          if (k0 <= qw0 + 31)  // some query of this wave sees it
            part(k0, t, t + P::kTile, 32 * i, [] {}, [] {});
        }
      };
      at_walk<P>((min(t0 + P::kOwn, len) - 1) / P::kRows + 1, smem, odd, fetch, compute);
    } else {
      E *Ks = reinterpret_cast<E*>(smem) + w * P::kTile, *Vs = reinterpret_cast<E*>(odd) + w * P::kTile;
      const int last = t0 / 32;
      if (w <= last) {
        at_load<E, HD, KS, VEC>(Vs, rows_of(vb, 32 * w), 0, lane);
        at_load<E, HD, KS, VEC>(Ks, rows_of(kb, 32 * w), 0, lane);
      }
      for (int p = w; p <= last; p += 4) {  // (past the last part nothing is in reach, and zeros arrive)
        at_wait<P::kLoads>();
        part(32 * p, Ks, Vs, 0,
             [&] {
               at_wait<-1>();
               at_load<E, HD, KS, VEC>(Vs, rows_of(vb, 32 * (p + 4)), 0, lane);
             },
             [&] { at_wait<P::kLoads>(); });
        at_wait<-1>();
        at_load<E, HD, KS, VEC>(Ks, rows_of(kb, 32 * (p + 4)), 0, lane);
      }
    }
  }
  E* dst = static_cast<E*>(a.dqkv) + row0 * a.qkv_cols + (size_t)h * a.hd;
  if constexpr (KS == 1) {
    at_landed();  // the tiles' LDS is free
    if (qw0 >= a.T) return;
    at_store<E, HD, VEC, P::kStaged>(dst + (size_t)qw0 * a.qkv_cols, a.qkv_cols, dq, a.scale, a.T - qw0, len - qw0, a.hd,
                         reinterpret_cast<E*>(smem) + w * 32 * HD, lane);
  } else {
    join_store<E, HD>(reinterpret_cast<float*>(smem), dq, a.scale, dst, t0, len, a.T, a.qkv_cols, a.hd, w, lane, tid);
  }
}

template <typename E, int HD, int KS, bool VEC>
__global__ __launch_bounds__(256, HD == 128 ? 1 : 2) void k_attn_backward_kv(const AttnTrain a) {
  typedef AtMma<E, HD> M;
  typedef AtPlan<E, HD, KS, VEC> P;
  constexpr bool kAhead = sizeof(E) == 2 && HD <= 64;  // registers for the transposed operand before the exponentials
  constexpr int kJoin = KS == 4 ? kJoinFloats<HD> * 4 : 0, kHalf = P::kBytes / 2;
  // KS == 1: [Q, dO] tiles, and the same for odd steps; KS == 4: the waves' Q tiles, and their dO tiles
  constexpr int kFirst = KS == 1 ? P::kBytes : kHalf > kJoin ? kHalf : kJoin;
  __shared__ __align__(1024) char smem[kFirst], odd[KS == 4 ? kHalf : P::kBufs == 2 ? P::kBytes : 16];
  constexpr int kStats = KS == 4 ? 4 : P::kParts;  // a buffer's 32-row parts: the tile's, or the waves'
  __shared__ __align__(1024) float stat[kStats][64], stat_odd[KS == 4 ? 1 : kStats][64];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const AtBlock at = at_block(blockIdx.x, a.B * a.Hk, a.ragged);
  const int b = at.g / a.Hk, kvh = at.g % a.Hk, group = a.H / a.Hk;
  const int k0 = at.blk * P::kOwn, len = at_len(a, b);
  const int kw0 = k0 + (KS == 1 ? 32 * w : 0), key = kw0 + (lane & 31);
  const size_t row0 = (size_t)b * a.T;
  const E* seq = static_cast<const E*>(a.qkv) + row0 * a.qkv_cols;
  const float sl2 = a.scale * kLog2e;

  at_f32x16 dk[HD / 32], dv[HD / 32];
#pragma unroll
  for (int dt = 0; dt < HD / 32; dt++) {
    at_zero(dk[dt]);
    at_zero(dv[dt]);
  }
  if (k0 < len) {
    const int n = min(32, len - kw0);
    const E* kb = seq + (size_t)kw0 * a.qkv_cols + (size_t)(a.H + kvh) * a.hd;
    const typename M::Own ko = M::template own<VEC>(at_rows(kb, n, a.qkv_cols, a.hd), lane & 31, lane);
    const typename M::Own vo =
        M::template own<VEC>(at_rows(kb + (size_t)a.Hk * a.hd, n, a.qkv_cols, a.hd), lane & 31, lane);
    const int head0 = kvh * group;
    auto q_rows = [&](int g, int q0) {
      return at_rows(seq + (size_t)q0 * a.qkv_cols + (size_t)(head0 + g) * a.hd, min(P::kRows, len - q0), a.qkv_cols, a.hd);
    };
    auto do_rows = [&](int g, int q0) {
      return at_rows(static_cast<const E*>(a.dout) + (row0 + q0) * a.out_cols + (size_t)(head0 + g) * a.hd,
                     min(P::kRows, len - q0), a.out_cols, a.hd);
    };
    // a part's statistics into LDS (past the length: zeros, which no part that counts reads)
    auto load_stat = [&](float* to, int g, int q0) {
      const float* from = stat_part(a, (size_t)b * a.H + head0 + g, q0);
      if constexpr (VEC)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(at_rows(from, q0 < len ? 1 : 0, 64, 64).rsrc,
                                                 (__attribute__((address_space(3))) void*)to, 4, lane * 4, 0, 0, 0);
      else
        to[lane] = q0 < len ? from[lane] : 0.f;
    };
    // the 32 queries from r0 on, tile rows i0 ..; the calls come before the Q tile and the statistics are read,
    // and where the dO tile has been read for the last time.
    // bf16: the products start from the statistics, p = 2^(sl2 (s - lse / scale)), ds = p (dP - D).
    auto part = [&](int r0, const E* Qs, const E* Os, int i0, const float* sp, auto&& q_wait, auto&& do_read) {
      at_f32x16 s, dp;
      const float* st = sp + 4 * (lane >> 5);
      typename M::Cols oc;
      if constexpr (sizeof(E) == 4) {
        at_zero(dp);
        at_zero(s);
        M::rows(dp, M::load_rows(Os, i0, lane), vo);
        q_wait();
        M::rows(s, M::load_rows(Qs, i0, lane), ko);
      } else {
        q_wait();
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const float4 l = *reinterpret_cast<const float4*>(st + 8 * c), d = *reinterpret_cast<const float4*>(st + 32 + 8 * c);
          s[4 * c] = l.x, s[4 * c + 1] = l.y, s[4 * c + 2] = l.z, s[4 * c + 3] = l.w;
          dp[4 * c] = d.x, dp[4 * c + 1] = d.y, dp[4 * c + 2] = d.z, dp[4 * c + 3] = d.w;
        }
        M::rows(dp, M::load_rows(Os, i0, lane), vo);
        M::rows(s, M::load_rows(Qs, i0, lane), ko);
        if (kAhead) oc = M::load_cols(Os, i0, lane);
      }
#pragma unroll
      for (int c = 0; c < 4; c++) {
        float l4[4], d4[4];
        if constexpr (sizeof(E) == 4) {
          const float4 l = *reinterpret_cast<const float4*>(st + 8 * c), d = *reinterpret_cast<const float4*>(st + 32 + 8 * c);
          l4[0] = l.x, l4[1] = l.y, l4[2] = l.z, l4[3] = l.w;
          d4[0] = d.x, d4[1] = d.y, d4[2] = d.z, d4[3] = d.w;
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int r = 4 * c + e;
          if constexpr (sizeof(E) == 4) {
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sl2, l4[e]));
            dp[r] = s[r] * (dp[r] + d4[e]);
          } else {
            s[r] = __builtin_amdgcn_exp2f(s[r] * sl2);
            dp[r] = s[r] * dp[r];
          }
        }
      }
      if (r0 < kw0 + 31) {                             // the part crosses the diagonal
        const int first = key - r0 - 4 * (lane >> 5);  // at_row0 of the first query that sees the key
#pragma unroll
        for (int r = 0; r < 16; r++)
          if (at_row0(r) < first) s[r] = dp[r] = 0.f;
      }
      if (!kAhead) oc = M::load_cols(Os, i0, lane);
      M::cols(dv, oc, s, lane);
      do_read();
      M::cols(dk, M::load_cols(Qs, i0, lane), dp, lane);
    };
    const int tiles = (len - k0 + P::kRows - 1) / P::kRows;  // of a head
    if constexpr (KS == 1) {
      int fg = 0, fq = k0, q0 = k0;  // head and first row of the tile to be requested next; first row of this one
      auto fetch = [&](int, char* buf) {
        E* t = reinterpret_cast<E*>(buf);
        at_load<E, HD, KS, VEC>(t, q_rows(fg, fq), w, lane);
        at_load<E, HD, KS, VEC>(t + P::kTile, do_rows(fg, fq), w, lane);
        if (w < P::kParts) load_stat(buf == smem ? stat[w] : stat_odd[w], fg, fq + 32 * w);
        fq += P::kRows;
        if (fq >= len) {
          fq = k0;
          fg++;
        }
      };
      auto compute = [&](int, const char* buf) {
        const E* t = reinterpret_cast<const E*>(buf);
#pragma unroll
        for (int i = 0; i < P::kParts; i++) {
          const int r0 = q0 + 32 * i;
          if (r0 + 31 < kw0 || r0 >= len) continue;  // every query of it is before these keys, or past the length
          const float* sp = buf == smem ? stat[i] : stat_odd[i];
          part(r0, t, t + P::kTile, 32 * i, sp, [] {}, [] {});
        }
        q0 += P::kRows;
        if (q0 >= len) q0 = k0;
      };
      at_walk<P>(tiles * group, smem, odd, fetch, compute);
    } else {
      E *Qs = reinterpret_cast<E*>(smem) + w * P::kTile, *Os = reinterpret_cast<E*>(odd) + w * P::kTile;
      int g = 0, p = w;  // this wave's part: of all heads' parts every fourth
      while (p >= tiles && g < group) p -= tiles, g++;
      if (g < group) {
        at_load<E, HD, KS, VEC>(Os, do_rows(g, k0 + 32 * p), 0, lane);
        at_load<E, HD, KS, VEC>(Qs, q_rows(g, k0 + 32 * p), 0, lane);
        load_stat(stat[w], g, k0 + 32 * p);
      }
      while (g < group) {
        const int r0 = k0 + 32 * p;
        p += 4;
        while (p >= tiles && g < group) p -= tiles, g++;
        const int ng = min(g, group - 1), nq = g < group ? k0 + 32 * p : a.T;  // past the last part: no rows
        at_wait<P::kLoads + 1>();
        part(r0, Qs, Os, 0, stat[w], [] { at_wait<0>(); },
             [&] {
               at_wait<-1>();
               at_load<E, HD, KS, VEC>(Os, do_rows(ng, nq), 0, lane);
             });
        at_wait<-1>();
        at_load<E, HD, KS, VEC>(Qs, q_rows(ng, nq), 0, lane);
        load_stat(stat[w], ng, nq);
      }
    }
  }
  E* dst = static_cast<E*>(a.dqkv) + row0 * a.qkv_cols + (size_t)(a.H + kvh) * a.hd;
  E* dstv = dst + (size_t)a.Hk * a.hd;
  if constexpr (KS == 1) {
    at_landed();  // the tiles' LDS is free
    if (kw0 >= a.T) return;
    E* tile = reinterpret_cast<E*>(smem) + w * 32 * HD;
    at_store<E, HD, VEC, P::kStaged>(dst + (size_t)kw0 * a.qkv_cols, a.qkv_cols, dk, a.scale, a.T - kw0, len - kw0, a.hd, tile, lane);
    at_store<E, HD, VEC, P::kStaged>(dstv + (size_t)kw0 * a.qkv_cols, a.qkv_cols, dv, 1.f, a.T - kw0, len - kw0, a.hd, tile, lane);
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
