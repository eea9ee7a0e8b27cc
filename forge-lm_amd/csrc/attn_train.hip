// attn_train.hip -- causal attention of packed q, k, v rows, forward (gfx950).
//
// Per (sequence, head), for a query i of the sequence's rows: s_ij = scale q_i . k_j for keys j <= i,
// o_i = sum_j exp(s_ij - lse_i) v_j with lse_i = log sum_j exp(s_ij).  One pass over the keys with a
// running maximum and sum; no score leaves the registers, and lse is all that the backward needs to
// compute the probabilities again.  Work: 4 hd operations a visible pair, q, k, v read and o written.
// Bound by the matrix cores and the exponentials beside them (32 x 32 scores of heads of 128: 512 cycles of
// products, some 480 of the softmax), small calls by latency.  Measured: 2 x 4096 bf16 rows, 16 heads of 128,
// 162 us (848 TFLOP/s); 4 x 512 fp32 rows, 12 heads of 64, 25 us (64 TFLOP/s); 8 x up to 777 bf16 rows 16.5 us.
#include "attn_train.hpp"

#include <math.h>

namespace fh {

namespace {

// at_spoilt: the rows of head h from t0 on, a lane's from its maximum and sum (base 2).
template <typename O, int HD>
__device__ __forceinline__ void forward_again(const AttnTrain& a, int b, int h, int t0, int len, float m, float l, int lane) {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // the stores before
  const O* x = static_cast<const O*>(a.qkv) + (size_t)b * a.T * a.qkv_cols;
  const O *k = x + (size_t)(a.H + h / (a.H / a.Hk)) * a.hd, *v = k + (size_t)a.Hk * a.hd;
  const int q = t0 + (lane & 31), d0 = (lane >> 5) * (HD / 2);
  if (t0 >= len || !at_hidden<O, false>(v + (size_t)t0 * a.qkv_cols, a.qkv_cols, min(32, len - t0), lane & 31, d0, HD / 2, a.hd))
    return;
  if (q >= len) return;
  const O* qr = x + (size_t)q * a.qkv_cols + (size_t)h * a.hd;
  float acc[HD / 2] = {};
#pragma unroll 1
  for (int j = 0; j <= q; j++) {
    const float p = __builtin_amdgcn_exp2f(fmaf(at_dot(qr, k + (size_t)j * a.qkv_cols, a.hd), a.scale * kLog2e, -m));
    at_add_row(acc, p, v + (size_t)j * a.qkv_cols, d0, a.hd);
  }
  at_put_row(static_cast<O*>(a.out) + ((size_t)b * a.T + q) * a.out_cols + (size_t)h * a.hd, acc, 1.f / l, d0, a.hd);
}

template <typename K, int HD, int KS, bool VEC>
__global__ __launch_bounds__(256, K::kParts * HD * KS >= 512 && sizeof(typename K::O) == 4 ? 1 : 2) void k_attn_forward(
    const AttnTrain a) {
  typedef AtMma<K, HD> M;
  typedef typename K::E E;
  typedef typename K::O O;
  typedef AtPlan<K, HD, KS, VEC> P;
  constexpr int N = HD < 64 ? HD : 64;  // dims joined at a time
  // V from memory to registers: a wave's own tile is read once, and its LDS is what a third block of the CU needs
  // (4 x 512 rows, 12 heads of 64: 35.3 and 31.6 us)
  constexpr bool kDirect = std::is_same_v<K, AtF32> && KS == 4 && HD <= 64;
  constexpr int kJoin = KS == 4 ? 4 * 32 * (N + 3) * 4 : 0, kHalf = P::kBytes / 2;
  // KS == 1: [K, V] tiles, and the same for odd steps; KS == 4: the waves' K tiles, and their V tiles
  constexpr int kFirst = KS == 1 ? P::kBytes : kHalf > kJoin ? kHalf : kJoin;
  __shared__ __align__(1024) char smem[kFirst], odd[kDirect ? 16 : KS == 4 ? kHalf : P::kBufs == 2 ? P::kBytes : 16];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nqb = (a.T + P::kOwn - 1) / P::kOwn;
  const AtBlock at = at_block(blockIdx.x, gridDim.x, 0, a.B * a.H, a.ragged);
  const int b = at.g / a.H, h = at.g % a.H, kvh = h / (a.H / a.Hk);
  const int t0 = (nqb - 1 - at.blk) * P::kOwn, len = at_len(a, b);
  const int qw0 = t0 + (KS == 1 ? 32 * w : 0), q = qw0 + (lane & 31);
  const AtSource<K> x = at_qkv<K>(a);
  const size_t row0 = (size_t)b * a.T;
  const int qc = h * a.in_hd, kc = (a.H + kvh) * a.in_hd, vc = kc + a.Hk * a.in_hd;  // columns
  const float sl2 = a.scale * kLog2e;
  at_f32x16 o[HD / 32];
#pragma unroll
  for (int dt = 0; dt < HD / 32; dt++) at_zero(o[dt]);
  float m = -INFINITY, l = 0.f;  // running maximum of scale * log2(e) * s, and sum

  if (t0 < len) {
    typename M::Own own;
    at_own<K, HD, VEC>(own, x, row0 + qw0, qc, min(32, len - qw0), lane);
    auto load = [&](E* tile, int col, int k0, int wave) {
      at_load<K, HD, KS, VEC>(tile, x, row0 + k0, col, len - k0, wave, lane);
    };
    // the 32 N keys from k0 on, tile rows r0 ..; the calls come where the K tile has been read for the last
    // time, and before the V tile is read
    auto part = [&](auto nparts, int k0, const E* Ks, const auto& V, int r0, auto&& k_read, auto&& v_wait) {
      constexpr int N = decltype(nparts)::value;
      at_f32x16 s[N];
      std::conditional_t<kDirect, char, typename M::Cols> vf[N];
#pragma unroll
      for (int i = 0; i < N; i++) {
        at_zero(s[i]);
        M::rows(s[i], Ks, P::kSub, r0 + 32 * i, own, lane);
      }
      k_read();
      v_wait();
      if constexpr (!kDirect)
#pragma unroll
        for (int i = 0; i < N; i++) vf[i] = M::load_cols(V, P::kSub, r0 + 32 * i, lane);
      const bool edge = N == 1 && k0 + 31 > qw0;  // the part crosses the diagonal
      if (edge) {
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
      if constexpr (kDirect)
        V.cols(o, s[0]);
      else
#pragma unroll
        for (int i = 0; i < N; i++) M::cols(o, vf[i], s[i], lane);
    };
    if constexpr (KS == 1) {
      auto fetch = [&](int kt, char* buf) {
        E* t = reinterpret_cast<E*>(buf);
        load(t, kc, kt * P::kRows, w);
        load(t + P::kTile, vc, kt * P::kRows, w);
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
    } else if constexpr (kDirect) {
      E* Ks = reinterpret_cast<E*>(smem) + w * P::kTile;
      const int last = t0 / 32;
      if (w <= last) load(Ks, kc, 32 * w, 0);
      for (int p = w; p <= last; p += 4) {  // (past the last part nothing is in reach, and zeros arrive)
        AtColsF32<HD> v;
        v.load(x.rows(0, row0 + 32 * p, vc, min(32, len - 32 * p)), lane);
        at_wait<16 * HD / 32>();
        part(at_int<1>, 32 * p, Ks, v, 0,
             [&] {
               at_wait<-1>();
               load(Ks, kc, 32 * (p + 4), 0);
             },
             [] {});
      }
    } else {
      E *Ks = reinterpret_cast<E*>(smem) + w * P::kTile, *Vs = reinterpret_cast<E*>(odd) + w * P::kTile;
      const int last = t0 / 32;
      if (w <= last) {
        load(Ks, kc, 32 * w, 0);
        load(Vs, vc, 32 * w, 0);
      }
      for (int p = w; p <= last; p += 4) {  // (past the last part nothing is in reach, and zeros arrive)
        at_wait<P::kLoads>();
        part(at_int<1>, 32 * p, Ks, Vs, 0,
             [&] {
               at_wait<-1>();
               load(Ks, kc, 32 * (p + 4), 0);
             },
             [&] { at_wait<P::kLoads>(); });
        at_wait<-1>();
        load(Vs, vc, 32 * (p + 4), 0);
      }
    }
    l += __shfl_xor(l, 32, 64);
  }

  O* out = static_cast<O*>(a.out) + (row0 + t0) * a.out_cols + (size_t)h * a.hd;
  float* lse = a.lse + (size_t)at.g * a.T;
  if constexpr (KS == 1) {
    at_landed();  // the tiles' LDS is free
    if (qw0 >= a.T) return;
    const bool row = q < len;
    at_store<O, HD, VEC, P::kOut>(out + (size_t)32 * w * a.out_cols, a.out_cols, o, row ? 1.f / l : 0.f, a.T - qw0, len - qw0,
                                   a.hd, reinterpret_cast<O*>(smem) + w * P::kOut * HD, lane);
    if (lane < 32 && q < a.T) lse[q] = row ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
    if (at_spoilt(o)) forward_again<O, HD>(a, b, h, qw0, len, m, l, lane);
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
        out[(size_t)i * a.out_cols + d0 + d] = (O)(t0 + i < len ? v / sum : 0.f);
      }
    }
    if (tid < 32 && t0 + tid < a.T) {
      const float sum = ol[tid] + ol[32 + tid] + ol[64 + tid] + ol[96 + tid];
      lse[t0 + tid] = t0 + tid < len ? (mx + __builtin_amdgcn_logf(sum)) * kLn2 : -INFINITY;
    }
    const int i = lane & 31;
    const float sum = ol[i] + ol[32 + i] + ol[64 + i] + ol[96 + i];
    if (at_block_spoilt(at_spoilt(o)) && w == 0) forward_again<O, HD>(a, b, h, t0, len, mx, sum, lane);
  }
}

// A matrix and where its parts go.
struct Split {
  const float* x;
  int cols, NH;  // columns of x's rows, heads
  __bf16* parts;
  size_t part;     // elements of one part
  const float* o;  // not null: x is do, and the rows' statistics are written too (stat_part)
  int blocks;
};
// The parts of NH heads of hd columns each of x's rows: rows of NH * hp columns of bf16, hp = hd to the next 8,
// zeros past hd; the three parts `part` elements apart.  A power of two of lanes, 1 << lg >= hp / 8, takes a
// row of a head.  Rows past a sequence's length are not read and not written.  The first blocks take s0, the
// others s1.
__global__ __launch_bounds__(256) void k_attn_split(const AttnTrain a, const Split s0, const Split s1, int lg) {
  const bool second = (int)blockIdx.x >= s0.blocks;
  const float *x = second ? s1.x : s0.x, *o = second ? s1.o : s0.o;
  const int x_cols = second ? s1.cols : s0.cols, NH = second ? s1.NH : s0.NH;
  __bf16* parts = second ? s1.parts : s0.parts;
  const size_t part = second ? s1.part : s0.part;
  const int block = blockIdx.x - (second ? s0.blocks : 0), blocks = second ? s1.blocks : s0.blocks;
  const int hp = a.in_hd, j = threadIdx.x & ((1 << lg) - 1), rows = a.T + 31 & ~31;
  const size_t n = (size_t)a.B * rows * NH;
  for (size_t i = ((size_t)block * 256 + threadIdx.x) >> lg; i < n; i += (size_t)blocks * (256 >> lg)) {
    const int h = i % NH, t = i / NH % rows, b = i / NH / rows, len = a.ragged ? (a.lens_dev ? a.lens_dev[b] : a.lens[b]) : a.T;
    const size_t row = (size_t)b * a.T + t;
    float v[8] = {}, D = 0.f;
    if (t < len && 8 * j < hp) {
      const float* from = x + row * x_cols + (size_t)h * a.hd + 8 * j;
      const float4 p = *reinterpret_cast<const float4*>(from);  // (hd is a multiple of 4)
      v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w;
      if (8 * j + 4 < a.hd) {
        const float4 q = *reinterpret_cast<const float4*>(from + 4);
        v[4] = q.x, v[5] = q.y, v[6] = q.z, v[7] = q.w;
      }
      if (o) {
        const float* of = o + row * a.out_cols + (size_t)h * a.hd + 8 * j;
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (8 * j + e < a.hd) D = fmaf(v[e], of[e], D);
      }
      __bf16* to = parts + row * ((size_t)NH * hp) + (size_t)h * hp + 8 * j;
#pragma unroll
      for (int p = 0; p < 3; p++) {
        at_bf16x8 b8;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          b8[e] = (__bf16)v[e];
          if (fabsf((float)b8[e]) == INFINITY)  // the largest values would round to it; an infinity is all here
            b8[e] = __builtin_bit_cast(__bf16, (unsigned short)(__float_as_uint(v[e]) >> 16));
          const float left = v[e] - (float)b8[e];
          v[e] = left == left ? left : 0.f;
        }
        *reinterpret_cast<at_bf16x8*>(to + p * part) = b8;
      }
    }
    if (o) {
      for (int s = 1; s < 1 << lg; s <<= 1) D += __shfl_xor(D, s, 64);
      const size_t head = (size_t)b * NH + h;
      if (j == 0) {
        float* st = a.stats + (head * (rows / 32) + t / 32) * 64 + t % 32;
        st[0] = t < len ? -a.lse[head * a.T + t] * kLog2e : -INFINITY;
        st[32] = t < len ? -D : 0.f;
      }
    }
  }
}

// Whether `blocks` blocks of 128 rows are so few that KS 4 pays: a wave's chain of steps is a quarter as long,
// and every tile is fetched for 32 rows instead of 128.  Fewer in bf16 where T is short: its chains cost little
// beside the join.  us with KS 1 and KS 4, 12 heads of 64 but where said:
//   bf16  192 blocks (2 x 1024) 20 and 16, 256 (4 x 1024, 8 heads) 21 and 23, 384 (4 x 1024) 24 and 29; heads of 32:
//         256 (2 x 1024, 16 heads) 17 and 14; shorter T: 96 (2 x 512) 11.1 and 9.9, 192 (4 x 512) 12.3 and 12.2, (8 x
//         256) 8.3 and 10, (16 x 128) 6.6 and 8.7; heads of 128: 96 (2 x 700, 8 heads) 22 and 17, 192 (4 x 400) 16 and 23
//   fp32  192 blocks 87 and 53, 384 100 and 89, 768 153 and 165; heads of 128: 256 blocks (2 x 2000, 8 heads) 291
//         and 228, 384 (8 x 300, 16 heads) 73 and 98
template <typename K, int HD>
bool few_blocks(size_t blocks, int T, int cus) {
  if (std::is_same_v<K, AtF32>) return 4 * blocks < (HD > 64 ? 5 : 8) * (size_t)cus;
  return 4 * 1024 * blocks < (HD > 32 ? 4 : 5) * (size_t)cus * (T < 1024 ? T : 1024);
}

template <typename K, int HD, bool VEC>
void forward_hd(hipStream_t st, const AttnTrain& a, int cus) {
  const size_t g = (size_t)a.B * a.H, wide = (size_t)((a.T + 127) / 128) * g, narrow = (size_t)((a.T + 31) / 32) * g;
  if constexpr (VEC && K::kParts == 1) {  // (parts: where blocks are many, attn_train_split)
    if (few_blocks<K, HD>(wide, a.T, cus)) {
      hipLaunchKernelGGL((k_attn_forward<K, HD, 4, VEC>), dim3((unsigned)narrow), dim3(256), 0, st, a);
      return;
    }
  }
  hipLaunchKernelGGL((k_attn_forward<K, HD, 1, VEC>), dim3((unsigned)wide), dim3(256), 0, st, a);
}

template <typename K, bool VEC>
void forward(hipStream_t st, const AttnTrain& a, int cus) {
  if (a.hd <= 32)
    forward_hd<K, 32, VEC>(st, a, cus);
  else if (a.hd <= 64)
    forward_hd<K, 64, VEC>(st, a, cus);
  else if constexpr (K::kParts == 1)
    forward_hd<K, 128, VEC>(st, a, cus);
}

// whether every row of a head can be moved by 16 bytes
bool whole_chunks(const AttnTrain& a, int esize) {
  auto ok = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
  const int n = 16 / esize;
  return a.hd % n == 0 && a.qkv_cols % n == 0 && a.out_cols % n == 0 && ok(a.qkv) && ok(a.out) && ok(a.dout) && ok(a.dqkv);
}

}  // namespace

// (of the launches, the largest has a block for every 32 rows of every head of q and of k and v: below 2^24)
bool attn_train_fits(const AttnTrain& a) {
  return a.B > 0 && a.B < 1 << 24 && a.T > 0 && a.Hk > 0 && a.H > 0 && a.H % a.Hk == 0 && a.hd > 0 && a.hd <= kAttnTrainHead &&
         a.T <= 1 << 24 && a.qkv_cols <= 1 << 20 && a.out_cols <= 1 << 20 &&
         (size_t)a.B * (a.H + a.Hk) * ((a.T + 31) / 32) < 1u << 24;
}

namespace {
size_t stat_floats(const AttnTrain& a) { return (size_t)a.B * a.H * ((a.T + 31) / 32) * 64; }
}  // namespace

// Whether fp32 tensors are multiplied in three bf16 parts, which takes 3/8 of the matrix cores' time and a launch
// that writes the parts.  12 heads of 64, us with the fp32 instruction and in parts:
//   forward   8 x 512 58 and 58, 16 x 512 90 and 91, 32 x 256 61 and 76; 4 x 1024 89 and 81, 8 x 1024 153 and
//             121, 2 x 2048 146 and 122; in few blocks 2 x 1024 53 and 70, 1 x 2048 84 and 93
//   backward  2 x 512 60 and 68, 2 x 700 85 and 91, 16 x 256 103 and 108; 4 x 512 96 and 84, 8 x 512 176 and 147,
//             1 x 1024 105 and 89, 4 x 1024 266 and 210, 8 x 1024 470 and 342, 1 x 2048 252 and 205
// Heads above 64 would not keep their three parts in registers.
bool attn_train_split(const AttnTrain& a, bool backward, int cus) {
  const size_t blocks = (size_t)a.B * a.H * ((a.T + 127) / 128);
  if (a.hd > 64 || !whole_chunks(a, 4)) return false;
  return backward ? a.T >= 1024 || (a.T > 256 && 4 * blocks >= 3 * (size_t)cus) : a.T > 512 && blocks > (size_t)cus;
}

size_t attn_train_scratch(const AttnTrain& a, bool bf16, bool backward, bool split, int cus) {
  const size_t stats = backward ? stat_floats(a) * 4 : 0;
  if (bf16 || !split || !attn_train_split(a, backward, cus)) return stats;
  const size_t hp = (a.hd + 7) / 8 * 8, rows = (size_t)a.B * a.T;
  return stats + 6 * rows * hp * (a.H + 2 * a.Hk + (backward ? a.H : 0));
}

// Fills what the kernels read: the tensors, or their parts, which are made first.
hipError_t attn_train_inputs(hipStream_t st, AttnTrain& a, bool bf16, bool backward, size_t scratch_bytes, int cus, bool* split,
                             bool* vec) {
  *vec = whole_chunks(a, bf16 ? 2 : 4);
  a.in = a.qkv, a.in_cols = a.qkv_cols, a.in_hd = a.hd, a.in_do = a.dout, a.do_cols = a.out_cols;
  a.in_part = a.do_part = 0;
  a.stats = static_cast<float*>(a.scratch);
  *split = !bf16 && attn_train_split(a, backward, cus) && scratch_bytes >= attn_train_scratch(a, bf16, backward, true, cus);
  if (!*split) return hipSuccess;
  const size_t rows = (size_t)a.B * a.T;
  a.in_hd = (a.hd + 7) / 8 * 8;
  a.in_cols = (a.H + 2 * a.Hk) * a.in_hd, a.do_cols = a.H * a.in_hd;
  a.in_part = rows * a.in_cols, a.do_part = rows * a.do_cols;
  __bf16* parts = reinterpret_cast<__bf16*>(a.stats + (backward ? stat_floats(a) : 0));
  __bf16* do_parts = parts + 3 * a.in_part;
  a.in = parts, a.in_do = do_parts;
  int lg = 0;
  while ((8 << lg) < a.in_hd) lg++;
  auto split_of = [&](const void* x, int cols, int heads, __bf16* to, size_t part, const void* o) {
    const size_t n = ((size_t)a.B * ((a.T + 31) / 32 * 32) * heads << lg) / 256 + 1;
    return Split{static_cast<const float*>(x), cols, heads, to, part, static_cast<const float*>(o),
                 (int)(n < 65536 ? n : 65536)};
  };
  const Split s0 = split_of(a.qkv, a.qkv_cols, a.H + 2 * a.Hk, parts, a.in_part, nullptr);
  Split s1{};
  if (backward) s1 = split_of(a.dout, a.out_cols, a.H, do_parts, a.do_part, a.out);
  hipLaunchKernelGGL(k_attn_split, dim3((unsigned)(s0.blocks + s1.blocks)), dim3(256), 0, st, a, s0, s1, lg);
  return hipGetLastError();
}

hipError_t launch_attn_forward(hipStream_t st, AttnTrain a, bool bf16, size_t scratch_bytes, int cus) {
  if (!attn_train_fits(a) || !a.qkv || !a.out || !a.lse) return hipErrorInvalidValue;
  bool split, vec;
  const hipError_t e = attn_train_inputs(st, a, bf16, false, a.scratch ? scratch_bytes : 0, cus, &split, &vec);
  if (e != hipSuccess) return e;
  if (split)
    forward<AtSplit, true>(st, a, cus);
  else if (bf16)
    vec ? forward<AtBf16, true>(st, a, cus) : forward<AtBf16, false>(st, a, cus);
  else
    vec ? forward<AtF32, true>(st, a, cus) : forward<AtF32, false>(st, a, cus);
  return hipGetLastError();
}

}  // namespace fh
