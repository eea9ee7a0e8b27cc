// attn_train_bwd.hip -- the backward pass of attn_train.hip, which computes the probabilities again
// from the scores and the forward's lse (gfx950).
//
//   p_ij = exp(scale q_i . k_j - lse_i)   D_i = do_i . o_i        ds_ij = p_ij (do_i . v_j - D_i)
//   dv_j = sum_i p_ij do_i                dq_i = scale sum_j ds_ij k_j   dk_j = scale sum_i ds_ij q_i
// Blocks of queries walk the keys (dq), blocks of keys the queries of every head that shares them (dk, dv),
// in one launch or in turn (backward_hd).  The scores and dP are computed in both, 14 hd operations a visible
// pair where 10 would do, so that every gradient is summed by one block in a fixed order: no atomics, the same
// bits on every run.  Bound by the matrix cores, the exponentials and products of a part beside them, and the
// chain of the longest blocks.  Measured, 12 heads of 64 (of the 14 hd operations): fp32 4 x 512 rows 69 us
// (82 TFLOP/s), 1 x 2500 238 us (141), bf16 8 x 1024 66 us (684).
#include "attn_train.hpp"

#include <math.h>

namespace fh {

hipError_t attn_train_inputs(hipStream_t st, AttnTrain& a, bool bf16, bool backward, size_t scratch_bytes, int cus, bool* split,
                             bool* vec);

namespace {

// The sum over the four waves of acc^T (dims x the 32 own rows), times f, to rows row0 .. of dst;
// rows at or past len are zeros, rows at or past T are not written.  os: kJoinFloats<HD>.
template <int HD>
constexpr int kJoinFloats = 4 * 32 * ((HD < 64 ? HD : 64) + 1);  // 64 dims at a time
template <typename O, int HD>
__device__ __forceinline__ void join_store(float* os, const at_f32x16 (&acc)[HD / 32], float f, O* dst, int row0, int len,
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
      dst[(size_t)(row0 + i) * stride + d0 + d] = (O)(row0 + i < len ? v * f : 0.f);
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

// p and ds of query i and key j, as the kernels have them
template <typename O>
__device__ __forceinline__ void score_again(const AttnTrain& a, int b, int h, int i, int j, float& p, float& ds) {
  const O* x = static_cast<const O*>(a.qkv) + (size_t)b * a.T * a.qkv_cols;
  const O* k = x + (size_t)j * a.qkv_cols + (size_t)(a.H + h / (a.H / a.Hk)) * a.hd;
  const size_t orow = ((size_t)b * a.T + i) * a.out_cols + (size_t)h * a.hd, head = (size_t)b * a.H + h;
  const O* dout = static_cast<const O*>(a.dout) + orow;
  const float D = at_dot(dout, static_cast<const O*>(a.out) + orow, a.hd);
  p = __builtin_amdgcn_exp2f(
      fmaf(at_dot(x + (size_t)i * a.qkv_cols + (size_t)h * a.hd, k, a.hd), a.scale * kLog2e, -a.lse[head * a.T + i] * kLog2e));
  ds = p * (at_dot(dout, k + (size_t)a.Hk * a.hd, a.hd) - D);
}
// at_spoilt: dq of the rows from t0 on.
template <typename O, int HD>
__device__ __forceinline__ void backward_q_again(const AttnTrain& a, int b, int h, int t0, int len, int lane) {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // the stores before
  const O* k = static_cast<const O*>(a.qkv) + (size_t)b * a.T * a.qkv_cols + (size_t)(a.H + h / (a.H / a.Hk)) * a.hd;
  const int q = t0 + (lane & 31), d0 = (lane >> 5) * (HD / 2);
  if (t0 >= len || !at_hidden<O, false>(k + (size_t)t0 * a.qkv_cols, a.qkv_cols, min(32, len - t0), lane & 31, d0, HD / 2, a.hd))
    return;
  if (q >= len) return;
  float acc[HD / 2] = {};
#pragma unroll 1
  for (int j = 0; j <= q; j++) {
    float p, ds;
    score_again<O>(a, b, h, q, j, p, ds);
    at_add_row(acc, ds, k + (size_t)j * a.qkv_cols, d0, a.hd);
  }
  at_put_row(static_cast<O*>(a.dqkv) + ((size_t)b * a.T + q) * a.qkv_cols + (size_t)h * a.hd, acc, a.scale, d0, a.hd);
}
// at_spoilt: dk and dv of the rows from k0 on.
template <typename O, int HD>
__device__ __forceinline__ void backward_kv_again(const AttnTrain& a, int b, int kvh, int k0, int len, int lane) {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // the stores before
  const int group = a.H / a.Hk, key = k0 + (lane & 31), d0 = (lane >> 5) * (HD / 2);
  const size_t row0 = (size_t)b * a.T;
  auto from = [&](int which, int h, int i) {  // a row of q or do
    return which ? static_cast<const O*>(a.dout) + (row0 + i) * a.out_cols + (size_t)h * a.hd
                 : static_cast<const O*>(a.qkv) + (row0 + i) * a.qkv_cols + (size_t)h * a.hd;
  };
#pragma unroll 1
  for (int which = 0; which < 2; which++) {  // dk, dv
    bool need = false;
#pragma unroll 1
    for (int h = kvh * group; h < (kvh + 1) * group && k0 < len; h++)
      need = need || at_hidden<O, true>(from(which, h, k0), which ? a.out_cols : a.qkv_cols, min(32, len - k0), lane & 31, d0,
                                        HD / 2, a.hd);
    if (!need || key >= len) continue;
    float acc[HD / 2] = {};
#pragma unroll 1
    for (int h = kvh * group; h < (kvh + 1) * group; h++)
#pragma unroll 1
      for (int i = key; i < len; i++) {
        float p, ds;
        score_again<O>(a, b, h, i, key, p, ds);
        at_add_row(acc, which ? p : ds, from(which, h, i), d0, a.hd);
      }
    O* to = static_cast<O*>(a.dqkv) + (row0 + key) * a.qkv_cols + (size_t)(a.H + kvh + (which ? a.Hk : 0)) * a.hd;
    at_put_row(to, acc, which ? 1.f : a.scale, d0, a.hd);
  }
}

// LDS of a block: two buffers that the walk tells apart by name, and for dk and dv the queries' statistics.
// KS == 1: a step's two tiles, and those of odd steps; KS == 4: the waves' tiles of one operand, and of the other.
template <typename K, int HD, int KS, bool VEC>
struct BackLds {
  typedef AtPlan<K, HD, KS, VEC> P;
  static constexpr int kJoin = KS == 4 ? kJoinFloats<HD> * 4 : 0, kHalf = P::kBytes / 2;
  static constexpr int kFirst = KS == 1 ? P::kBytes : kHalf > kJoin ? kHalf : kJoin;
  static constexpr int kOdd = KS == 4 ? kHalf : P::kBufs == 2 ? P::kBytes : 16;
  static constexpr int kStats = KS == 4 ? 4 : P::kParts, kStatsOdd = KS == 4 ? 1 : P::kParts;  // 32-row parts
};

// dq of block `block` of `blocks`.  STATS: the statistics are there; else this computes them for the other kernel.
template <typename K, int HD, int KS, bool VEC, bool STATS>
__device__ __forceinline__ void backward_q(const AttnTrain& a, int block, int blocks, int before, char* smem, char* odd) {
  typedef AtMma<K, HD> M;
  typedef typename K::E E;
  typedef typename K::O O;
  typedef AtPlan<K, HD, KS, VEC> P;

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nqb = (a.T + P::kOwn - 1) / P::kOwn;
  const AtBlock at = at_block(block, blocks, before, a.B * a.H, a.ragged);
  const int b = at.g / a.H, h = at.g % a.H, kvh = h / (a.H / a.Hk);
  const int t0 = (nqb - 1 - at.blk) * P::kOwn, len = at_len(a, b);
  const int qw0 = t0 + (KS == 1 ? 32 * w : 0), q = qw0 + (lane & 31);
  const size_t row0 = (size_t)b * a.T;
  const AtSource<K> x = at_qkv<K>(a), xo = at_do<K>(a);
  const int qc = h * a.in_hd, kc = (a.H + kvh) * a.in_hd, vc = kc + a.Hk * a.in_hd;  // columns
  const float sl2 = a.scale * kLog2e;

  at_f32x16 dq[HD / 32];
#pragma unroll
  for (int dt = 0; dt < HD / 32; dt++) at_zero(dq[dt]);

  if (t0 < len) {
    const int n = min(32, len - qw0);
    typename M::Own own, dout;
    at_own<K, HD, VEC>(own, x, row0 + qw0, qc, n, lane);
    at_own<K, HD, VEC>(dout, xo, row0 + qw0, qc, n, lane);
    std::conditional_t<STATS, char, typename M::Own> o;
    if constexpr (!STATS)
      at_own<K, HD, VEC>(o, AtSource<K>{static_cast<const E*>(a.out), 0, a.out_cols, a.hd}, row0 + qw0, qc, n, lane);
    // the first tiles are on their way while D waits for the rows above
    auto load = [&](E* tile, int col, int k0, int wave) {
      at_load<K, HD, KS, VEC>(tile, x, row0 + k0, col, len - k0, wave, lane);
    };
    auto fetch = [&](int kt, char* buf) {
      E* t = reinterpret_cast<E*>(buf);
      load(t, kc, kt * P::kRows, w);
      load(t + P::kTile, vc, kt * P::kRows, w);
    };
    E *Ks = reinterpret_cast<E*>(smem) + w * P::kTile, *Vs = reinterpret_cast<E*>(odd) + w * P::kTile;  // KS == 4
    const int last = t0 / 32;
    if constexpr (KS == 4) {
      if (w <= last) {
        load(Vs, vc, 32 * w, 0);
        load(Ks, kc, 32 * w, 0);
      }
    } else if constexpr (P::kBufs == 2) {
      fetch(0, smem);
    }
    float D, lse2;
    if constexpr (STATS) {
      const float* st = stat_part(a, at.g, qw0) + (lane & 31);
      lse2 = q < len ? sizeof(O) == 4 ? -st[0] : -st[0] * sl2 : INFINITY;
      D = q < len ? -st[32] : 0.f;
    } else {
      D = M::dot(dout.v[0], o.v[0]);
      D += __shfl_xor(D, 32, 64);
      lse2 = q < len ? a.lse[(size_t)at.g * a.T + q] * kLog2e : INFINITY;
      if ((KS == 1 || w == 0) && qw0 < len)
        stat_part(a, at.g, qw0)[lane] = lane >= 32 ? -D : sizeof(O) == 4 ? -lse2 : -lse2 / sl2;
    }
    // the 32 keys from k0 on, tile rows r0 ..; the calls come where the V tile has been read for the last
    // time, and before the K tile is read
    auto part = [&](int k0, const E* Ks, const E* Vs, int r0, auto&& v_read, auto&& k_wait) {
      at_f32x16 s, dp;
      at_zero(dp);
      M::rows(dp, Vs, P::kSub, r0, dout, lane);
      v_read();
      k_wait();
      at_zero(s);
      M::rows(s, Ks, P::kSub, r0, own, lane);
      const typename M::Cols kf = M::load_cols(Ks, P::kSub, r0, lane);
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sl2, -lse2)) * (dp[r] - D);
      if (k0 + 31 > qw0) {                          // the part crosses the diagonal
        const int left = q - k0 - 4 * (lane >> 5);  // at_row0 of the last key that the query sees
#pragma unroll
        for (int r = 0; r < 16; r++)
          if (at_row0(r) > left) s[r] = 0.f;
      }
      M::cols(dq, kf, s, lane);
    };
    if constexpr (KS == 1) {
      auto compute = [&](int kt, const char* buf) {
        const E* t = reinterpret_cast<const E*>(buf);
#pragma unroll
        for (int i = 0; i < P::kParts; i++) {
          const int k0 = kt * P::kRows + 32 * i;
          if (k0 <= qw0 + 31)  // some query of this wave sees it
            part(k0, t, t + P::kTile, 32 * i, [] {}, [] {});
        }
      };
      at_walk<P, P::kBufs == 2>((min(t0 + P::kOwn, len) - 1) / P::kRows + 1, smem, odd, fetch, compute);
    } else {
      for (int p = w; p <= last; p += 4) {  // (past the last part nothing is in reach, and zeros arrive)
        at_wait<P::kLoads>();
        part(32 * p, Ks, Vs, 0,
             [&] {
               at_wait<-1>();
               load(Vs, vc, 32 * (p + 4), 0);
             },
             [&] { at_wait<P::kLoads>(); });
        at_wait<-1>();
        load(Ks, kc, 32 * (p + 4), 0);
      }
    }
  }
  O* dst = static_cast<O*>(a.dqkv) + row0 * a.qkv_cols + (size_t)h * a.hd;
  if constexpr (KS == 1) {
    at_landed();  // the tiles' LDS is free
    if (qw0 >= a.T) return;
    at_store<O, HD, VEC, P::kOut>(dst + (size_t)qw0 * a.qkv_cols, a.qkv_cols, dq, a.scale, a.T - qw0, len - qw0, a.hd,
                                   reinterpret_cast<O*>(smem) + w * P::kOut * HD, lane);
    if (at_spoilt(dq)) backward_q_again<O, HD>(a, b, h, qw0, len, lane);
  } else {
    join_store<O, HD>(reinterpret_cast<float*>(smem), dq, a.scale, dst, t0, len, a.T, a.qkv_cols, a.hd, w, lane, tid);
    if (at_block_spoilt(at_spoilt(dq)) && w == 0) backward_q_again<O, HD>(a, b, h, t0, len, lane);
  }
}

// dk and dv of block `block` of `blocks`.
template <typename K, int HD, int KS, bool VEC>
__device__ __forceinline__ void backward_kv(const AttnTrain& a, int block, int blocks, char* smem, char* odd, float (*stat)[64],
                                            float (*stat_odd)[64]) {
  typedef AtMma<K, HD> M;
  typedef typename K::E E;
  typedef typename K::O O;
  typedef AtPlan<K, HD, KS, VEC> P;

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const AtBlock at = at_block(block, blocks, 0, a.B * a.Hk, a.ragged);
  const int b = at.g / a.Hk, kvh = at.g % a.Hk, group = a.H / a.Hk;
  const int k0 = at.blk * P::kOwn, len = at_len(a, b);
  const int kw0 = k0 + (KS == 1 ? 32 * w : 0), key = kw0 + (lane & 31);
  const size_t row0 = (size_t)b * a.T;
  const AtSource<K> x = at_qkv<K>(a), xo = at_do<K>(a);
  const float sl2 = a.scale * kLog2e;

  at_f32x16 dk[HD / 32], dv[HD / 32];
#pragma unroll
  for (int dt = 0; dt < HD / 32; dt++) {
    at_zero(dk[dt]);
    at_zero(dv[dt]);
  }
  if (k0 < len) {
    const int n = min(32, len - kw0), kc = (a.H + kvh) * a.in_hd;
    typename M::Own ko, vo;
    at_own<K, HD, VEC>(ko, x, row0 + kw0, kc, n, lane);
    at_own<K, HD, VEC>(vo, x, row0 + kw0, kc + a.Hk * a.in_hd, n, lane);
    const int head0 = kvh * group;
    auto load = [&](E* tile, const AtSource<K>& m, int g, int q0, int wave) {
      at_load<K, HD, KS, VEC>(tile, m, row0 + q0, (size_t)(head0 + g) * a.in_hd, len - q0, wave, lane);
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
      if constexpr (sizeof(O) == 4) {
        at_zero(dp);
        at_zero(s);
        M::rows(dp, Os, P::kSub, i0, vo, lane);
        q_wait();
      } else {
        q_wait();
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const float4 l = *reinterpret_cast<const float4*>(st + 8 * c), d = *reinterpret_cast<const float4*>(st + 32 + 8 * c);
          s[4 * c] = l.x, s[4 * c + 1] = l.y, s[4 * c + 2] = l.z, s[4 * c + 3] = l.w;
          dp[4 * c] = d.x, dp[4 * c + 1] = d.y, dp[4 * c + 2] = d.z, dp[4 * c + 3] = d.w;
        }
        M::rows(dp, Os, P::kSub, i0, vo, lane);
      }
      M::rows(s, Qs, P::kSub, i0, ko, lane);
      const typename M::Cols of = M::load_cols(Os, P::kSub, i0, lane);
#pragma unroll
      for (int c = 0; c < 4; c++) {
        float l4[4], d4[4];
        if constexpr (sizeof(O) == 4) {
          const float4 l = *reinterpret_cast<const float4*>(st + 8 * c), d = *reinterpret_cast<const float4*>(st + 32 + 8 * c);
          l4[0] = l.x, l4[1] = l.y, l4[2] = l.z, l4[3] = l.w;
          d4[0] = d.x, d4[1] = d.y, d4[2] = d.z, d4[3] = d.w;
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int r = 4 * c + e;
          if constexpr (sizeof(O) == 4) {
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
      M::cols(dv, of, s, lane);
      do_read();
      M::cols(dk, M::load_cols(Qs, P::kSub, i0, lane), dp, lane);
    };
    const int tiles = (len - k0 + P::kRows - 1) / P::kRows;  // of a head
    if constexpr (KS == 1) {
      int fg = 0, fq = k0, q0 = k0;  // head and first row of the tile to be requested next; first row of this one
      auto fetch = [&](int, char* buf) {
        E* t = reinterpret_cast<E*>(buf);
        load(t, x, fg, fq, w);
        load(t + P::kTile, xo, fg, fq, w);
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
        load(Os, xo, g, k0 + 32 * p, 0);
        load(Qs, x, g, k0 + 32 * p, 0);
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
               load(Os, xo, ng, nq, 0);
             });
        at_wait<-1>();
        load(Qs, x, ng, nq, 0);
        load_stat(stat[w], ng, nq);
      }
    }
  }
  O* dst = static_cast<O*>(a.dqkv) + row0 * a.qkv_cols + (size_t)(a.H + kvh) * a.hd;
  O* dstv = dst + (size_t)a.Hk * a.hd;
  if constexpr (KS == 1) {
    at_landed();  // the tiles' LDS is free
    if (kw0 >= a.T) return;
    O* tile = reinterpret_cast<O*>(smem) + w * P::kOut * HD;
    at_store<O, HD, VEC, P::kOut>(dst + (size_t)kw0 * a.qkv_cols, a.qkv_cols, dk, a.scale, a.T - kw0, len - kw0, a.hd, tile, lane);
    at_store<O, HD, VEC, P::kOut>(dstv + (size_t)kw0 * a.qkv_cols, a.qkv_cols, dv, 1.f, a.T - kw0, len - kw0, a.hd, tile, lane);
    if (at_spoilt(dk) || at_spoilt(dv)) backward_kv_again<O, HD>(a, b, kvh, kw0, len, lane);
  } else {
    float* os = reinterpret_cast<float*>(smem);
    join_store<O, HD>(os, dk, a.scale, dst, k0, len, a.T, a.qkv_cols, a.hd, w, lane, tid);
    join_store<O, HD>(os, dv, 1.f, dstv, k0, len, a.T, a.qkv_cols, a.hd, w, lane, tid);
    if (at_block_spoilt(at_spoilt(dk) || at_spoilt(dv)) && w == 0) backward_kv_again<O, HD>(a, b, kvh, k0, len, lane);
  }
}

template <typename K, int HD, int KS, bool VEC>
__global__ __launch_bounds__(256, HD > 64 && sizeof(typename K::O) == 4 ? 1 : 2) void k_attn_backward_q(const AttnTrain a) {
  typedef BackLds<K, HD, KS, VEC> L;
  __shared__ __align__(1024) char smem[L::kFirst], odd[L::kOdd];
  backward_q<K, HD, KS, VEC, false>(a, blockIdx.x, gridDim.x, 0, smem, odd);
}
// Waves of dk and dv that a SIMD's registers hold at least (heads of 128, and parts of 64 where LDS has no room
// for more: one)
template <typename K, int HD, int KS>
constexpr int kWaves = HD > 64 || (HD > 32 && K::kParts > 1 && KS == 4) ? 1 : 2;
template <typename K, int HD, int KS, bool VEC>
__global__ __launch_bounds__(256, (kWaves<K, HD, KS>)) void k_attn_backward_kv(const AttnTrain a) {
  typedef BackLds<K, HD, KS, VEC> L;
  __shared__ __align__(1024) char smem[L::kFirst], odd[L::kOdd];
  __shared__ __align__(1024) float stat[L::kStats][64], stat_odd[L::kStatsOdd][64];
  backward_kv<K, HD, KS, VEC>(a, blockIdx.x, gridDim.x, smem, odd, stat, stat_odd);
}
// Both in one launch: the blocks of dk and dv first, which have more to do, and those of dq fill the CUs that
// the last of them leave idle.
template <typename K, int HD, int QS, int KS>
__global__ __launch_bounds__(256, (kWaves<K, HD, KS>)) void k_attn_backward_both(const AttnTrain a, int kv_blocks) {
  typedef BackLds<K, HD, KS, true> L;
  typedef BackLds<K, HD, QS, true> Q;
  __shared__ __align__(1024) char smem[L::kFirst > Q::kFirst ? L::kFirst : Q::kFirst], odd[L::kOdd > Q::kOdd ? L::kOdd : Q::kOdd];
  __shared__ __align__(1024) float stat[L::kStats][64], stat_odd[L::kStatsOdd][64];
  if ((int)blockIdx.x < kv_blocks)
    backward_kv<K, HD, KS, true>(a, blockIdx.x, kv_blocks, smem, odd, stat, stat_odd);
  else
    backward_q<K, HD, QS, true, true>(a, blockIdx.x - kv_blocks, gridDim.x - kv_blocks, kWaves<K, HD, KS> > 1 ? kv_blocks : 0, smem, odd);
}

// The rows' statistics (stat_part), 8 lanes to a row of a head.  Those of parts past a length are not read.
template <typename O>
__global__ __launch_bounds__(256) void k_attn_stats(const AttnTrain a) {
  constexpr int CE = 16 / sizeof(O);
  const int j = threadIdx.x & 7, rows = (a.T + 31) & ~31;
  const size_t n = (size_t)a.B * rows * a.H;
  for (size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) >> 3; i < n; i += (size_t)gridDim.x * 32) {
    const int h = i % a.H, t = i / a.H % rows, b = i / a.H / rows;
    const int len = a.ragged ? (a.lens_dev ? a.lens_dev[b] : a.lens[b]) : a.T;
    const size_t row = ((size_t)b * a.T + t) * a.out_cols + (size_t)h * a.hd;
    float D = 0.f;
    for (int c = j; c * CE < a.hd && t < len; c += 8) {  // (hd is a multiple of CE)
      typedef O oc __attribute__((ext_vector_type(CE)));
      const oc x = *reinterpret_cast<const oc*>(static_cast<const O*>(a.dout) + row + c * CE);
      const oc y = *reinterpret_cast<const oc*>(static_cast<const O*>(a.out) + row + c * CE);
#pragma unroll
      for (int e = 0; e < CE; e++) D = fmaf((float)x[e], (float)y[e], D);
    }
#pragma unroll
    for (int s = 1; s < 8; s <<= 1) D += __shfl_xor(D, s, 64);
    const size_t head = (size_t)b * a.H + h;
    if (j == 0) {
      float* st = stat_part(a, head, t) + t % 32;
      st[0] = t < len ? -a.lse[head * a.T + t] * (sizeof(O) == 4 ? kLog2e : 1.f / a.scale) : -INFINITY;
      st[32] = t < len ? -D : 0.f;
    }
  }
}

// Whether `blocks` blocks of 128 rows, which walk the rows of `heads` heads, are so few that KS 4 pays (chains a
// quarter as long, tiles fetched for 32 rows instead of 128); fewer where T is so short that a block of 128 rows
// has no chain.  us with KS 1 and KS 4, dq, dk and dv in one launch:
//   bf16, 12 heads of 64   96 blocks (1 x 1024) 29 and 25, (2 x 512) 19 and 21; 144 (3 x 512) 21 and 28; 192
//                          (2 x 1024) 34 and 39, (1 x 2048) 58 and 56; heads of 32: 128 (2 x 2048, 4 heads) 38 and
//                          24; heads of 128: 96 (1 x 700, 16 heads) 35 and 47
//   in parts               96 (1 x 1024) 110 and 88, 192 (2 x 1024) 129 and 155, 240 (1 x 2500) 271 and 309; heads
//                          of 32: 128 (2 x 2048, 4 heads) 130 and 82
//   fp32                   192 (4 x 512) 118 and 95, (8 x 256) 71 and 67, (16 x 128) 43 and 51; 288 (12 x 256) 80
//                          and 98; heads of 128: 128 (1 x 1000, 16 heads) 283 and 215, (8 x 128) 54 and 82
//   dk and dv where 4 heads share k and v (dq KS 1): bf16 64 blocks (4 x 1024, 8 heads of 64) 90 and 43, 176
//                          (4 x 1333, 16 heads of 128) 212 and 205
template <typename K, int HD>
bool few_blocks(size_t blocks, int T, int heads, int cus) {
  const int q = std::is_same_v<K, AtF32> ? HD > 64 ? 3 : 4 : HD > 64 ? 1 : HD > 32 ? 2 : 3;  // quarters of the CUs
  const int quarters = heads < q ? q : heads > 4 ? 4 : heads;
  return 4 * 256 * blocks < (size_t)quarters * cus * (T < 256 ? T : 256);
}

template <typename K, int HD, bool VEC>
void backward_hd(hipStream_t st, const AttnTrain& a, int cus) {
  const size_t wide = (size_t)((a.T + 127) / 128), narrow = (size_t)((a.T + 31) / 32);
  const size_t gq = (size_t)a.B * a.H, gk = (size_t)a.B * a.Hk;
  // dq in blocks of 128 rows, and then dk and dv
  auto in_turn = [&](auto ks) {
    constexpr int KS = decltype(ks)::value;
    hipLaunchKernelGGL((k_attn_backward_q<K, HD, 1, VEC>), dim3((unsigned)(wide * gq)), dim3(256), 0, st, a);
    hipLaunchKernelGGL((k_attn_backward_kv<K, HD, KS, VEC>), dim3((unsigned)((KS == 4 ? narrow : wide) * gk)), dim3(256), 0, st, a);
  };
  auto together = [&](auto qs, auto ks) {
    constexpr int QS = decltype(qs)::value, KS = decltype(ks)::value;
    const size_t kv = (KS == 4 ? narrow : wide) * gk, q = (QS == 4 ? narrow : wide) * gq;
    if constexpr (K::kParts == 1)
      hipLaunchKernelGGL((k_attn_stats<typename K::O>), dim3((unsigned)(narrow * gq)), dim3(256), 0, st, a);
    hipLaunchKernelGGL((k_attn_backward_both<K, HD, QS, KS>), dim3((unsigned)(kv + q)), dim3(256), 0, st, a, (int)kv);
  };
  if constexpr (!VEC) {
    in_turn(at_int<1>);
  } else {
    const bool few_q = few_blocks<K, HD>(wide * gq, a.T, 1, cus);
    const bool few_k = few_q || few_blocks<K, HD>(wide * gk, a.T, a.H / a.Hk, cus);
    if (few_q) {
      together(at_int<4>, at_int<4>);
      return;
    }
    // One launch costs the statistics' (3 to 5 us; with parts they come anyway), and bf16's dq the waves that the
    // registers of dk and dv leave no room for; it saves what the CUs idle while the last blocks of dk and dv end,
    // which are up to T / 128 times as long as the first.  us in turn and in one, by blocks of dk and dv:
    //   bf16, 12 heads of 64  384 (4 x 1024) 57 and 46, 384 (1 x 4096) 182 and 129, 768 (8 x 1024) 77 and 83
    //   bf16, 16 heads of 128  256 (2 x 4096, 4 of k and v) 761 and 652, 384 (8 x 300) 43 and 49; in blocks of 32
    //                  and dq in 704 (4 x 1333, 4 of k and v) 205 and 226, in 192 (4 x 700, 8 heads, 2) 69 and 53
    //   fp32, 12 heads of 64  768 (32 x 256) 189 and 174; in parts, 768 (16 x 512) 233 and 218, (8 x 1024) 336 and 318
    if constexpr (!std::is_same_v<K, AtBf16>) {
      few_k ? together(at_int<1>, at_int<4>) : together(at_int<1>, at_int<1>);
    } else if constexpr (HD <= 64) {
      if (few_k)
        together(at_int<1>, at_int<4>);
      else if (wide * gk < 2 * (size_t)cus)
        together(at_int<1>, at_int<1>);
      else
        in_turn(at_int<1>);
    } else {
      if (few_k)
        wide * gq <= 2 * (size_t)cus ? together(at_int<1>, at_int<4>) : in_turn(at_int<4>);
      else if (wide * gk <= (size_t)cus)
        together(at_int<1>, at_int<1>);
      else
        in_turn(at_int<1>);
    }
  }
}

template <typename K, bool VEC>
void backward(hipStream_t st, const AttnTrain& a, int cus) {
  if (a.hd <= 32)
    backward_hd<K, 32, VEC>(st, a, cus);
  else if (a.hd <= 64)
    backward_hd<K, 64, VEC>(st, a, cus);
  else if constexpr (K::kParts == 1)
    backward_hd<K, 128, VEC>(st, a, cus);
}

}  // namespace

hipError_t launch_attn_backward(hipStream_t st, AttnTrain a, bool bf16, size_t scratch_bytes, int cus) {
  if (!attn_train_fits(a) || !a.qkv || !a.out || !a.lse || !a.dout || !a.dqkv || !a.scratch ||
      scratch_bytes < attn_train_scratch(a, bf16, true, false, cus))
    return hipErrorInvalidValue;
  bool split, vec;
  const hipError_t e = attn_train_inputs(st, a, bf16, true, scratch_bytes, cus, &split, &vec);
  if (e != hipSuccess) return e;
  if (split)
    backward<AtSplit, true>(st, a, cus);
  else if (bf16)
    vec ? backward<AtBf16, true>(st, a, cus) : backward<AtBf16, false>(st, a, cus);
  else
    vec ? backward<AtF32, true>(st, a, cus) : backward<AtF32, false>(st, a, cus);
  return hipGetLastError();
}

}  // namespace fh
