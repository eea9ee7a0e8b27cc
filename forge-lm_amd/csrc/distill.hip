// distill.hip -- the loss of a student against a teacher's top logits and hard targets, and its
// gradient (gfx950).
//
// Row t, student logits z, teacher logits u_k for the ids i_k of its used slots, temperature tau:
//   q = softmax(u / tau) over the used slots      p = softmax(z / tau), p1 = softmax(z) over all V
//   loss_t = alpha tau^2 sum_k q_k (log q_k - log p_{i_k}) - (1 - alpha) log p1_target
//   dz_v   = [alpha tau (p_v - sum_{i_k = v} q_k) + (1 - alpha) (p1_v - [v = target])] / count
// With e = exp((z - max z) / tau) and f_k = exp((u_k - max u) / tau), the first sum is
// (sum_k f_k (u'_k - z'_k)) / sum f - log sum f + log sum e, so a row's maxima and its sums are all it
// needs.  HBM-bound: a row is read once into a block's registers and its gradient written from them;
// the K touched columns are written again after the dense ones (their sums in slot order: repeated
// ids add up in a fixed order).
#include "kernels.hpp"

#include <math.h>

namespace fh {

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The VW = 16 / sizeof(E) elements of a 16-byte vector, and back (rounded to nearest even).
template <typename E>
__device__ __forceinline__ float element(const u32x4& v, int e);
template <>
__device__ __forceinline__ float element<float>(const u32x4& v, int e) { return __uint_as_float(v[e]); }
template <>
__device__ __forceinline__ float element<bf16_t>(const u32x4& v, int e) {
  return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
}
template <typename E>
__device__ __forceinline__ u32x4 pack(const float* f);
template <>
__device__ __forceinline__ u32x4 pack<float>(const float* f) {
  return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
}
template <>
__device__ __forceinline__ u32x4 pack<bf16_t>(const float* f) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = __builtin_bit_cast(unsigned, b2{(__bf16)f[2 * i], (__bf16)f[2 * i + 1]});
  return v;
}

// max(a, b, c), a NaN only of three; one instruction where fmaxf also quiets what was loaded
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Sums (or the maximum of the first two) of N values over a block of BT threads; red: BT / 64 rows of N.
template <int BT, int N, bool MAX>
__device__ __forceinline__ void block_reduce(float (&v)[N], float (*red)[8]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = MAX ? wave_max_dpp(v[i]) : wave_sum_dpp(v[i]);
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; i++) red[w][i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = red[0][i];
#pragma unroll
  for (int j = 1; j < BT / 64; j++)
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = MAX ? fmaxf(v[i], red[j][i]) : v[i] + red[j][i];
}

// A row's exponents: 2^(z ct - mt) and, where a second exponential is needed, 2^(z c1 - m1).  mt is m ct
// rounded: what that leaves (rt, r1) is a factor of every exponential of the row, which the gradient does
// not see and the loss puts right.
struct RowExp {
  float ct, mt, rt, c1, m1, r1;
  bool two;
  __device__ __forceinline__ RowExp(const DistillArgs& a, float m) {
    two = a.alpha > 0.f && a.alpha < 1.f && a.tau != 1.f;  // (tau 1, or one of the two terms alone: one serves)
    ct = a.alpha > 0.f ? kLog2e / a.tau : kLog2e;
    c1 = kLog2e;
    mt = m * ct;
    rt = fmaf(m, ct, -mt);
    m1 = m * c1;
    r1 = fmaf(m, c1, -m1);
  }
  __device__ __forceinline__ float soft(float z) const { return __builtin_amdgcn_exp2f(fmaf(z, ct, -mt)); }
  __device__ __forceinline__ float hard(float z) const { return __builtin_amdgcn_exp2f(fmaf(z, c1, -m1)); }
};

// What a row's columns need once its sums are known.  bf16: the weights are in the exponents, whose
// roundings (2^-19 at most) are far below the gradient's.
template <typename E>
struct RowGrad {
  RowExp x;
  float at, a1;  // weights of the two exponentials (bf16: added to the exponents)
  __device__ __forceinline__ float operator()(float z) const {
    float g;
    if constexpr (sizeof(E) == 2) {
      g = __builtin_amdgcn_exp2f(fmaf(z, x.ct, at));
      if (x.two) g += __builtin_amdgcn_exp2f(fmaf(z, x.c1, a1));
    } else {
      g = at * x.soft(z);
      if (x.two) g = fmaf(a1, x.hard(z), g);
    }
    return g;
  }
};

// The row's loss and gradient weights from its sums.  sums: x.soft, x.hard, f, f u', f z'.
template <typename E>
__device__ __forceinline__ float row_loss(const DistillArgs& a, float m, const float (&sums)[5], float zt, RowGrad<E>& g) {
  const RowExp& x = g.x;
  const float st = sums[0], s1 = x.two ? sums[1] : sums[0], sf = sums[2];
  const bool kept = sf > 0.f || sf != sf;  // a row with a used slot (a NaN among them goes on)
  const float lt = (__builtin_amdgcn_logf(st) - x.rt) * kLn2;  // log of the sum of e
  const float l1 = x.two ? (__builtin_amdgcn_logf(s1) - x.r1) * kLn2 : lt;
  float loss = 0.f;
  if (a.alpha > 0.f && kept)
    loss = a.alpha * a.tau * a.tau * ((sums[3] - sums[4]) / sf + (lt - __builtin_amdgcn_logf(sf) * kLn2));
  if (a.alpha < 1.f) loss += (1.f - a.alpha) * (l1 - (zt - m));
  const float wt = kept ? a.alpha * a.tau * a.inv_count : 0.f, w1 = (1.f - a.alpha) * a.inv_count;
  g.at = (x.two ? wt : wt + w1) / st;
  g.a1 = w1 / s1;
  if (sizeof(E) == 2) {
    g.at = __builtin_amdgcn_logf(g.at) - x.mt;
    g.a1 = __builtin_amdgcn_logf(g.a1) - x.m1;
  }
  return loss;
}

// The teacher's slots of a row in LDS: ids (-1: empty) and f_k, and this thread's shares of the sums.
template <int BT>
__device__ __forceinline__ float load_slots(const DistillArgs& a, size_t row, int* ids, float* f) {
  float mu = -INFINITY;
  for (int k = threadIdx.x; k < a.K; k += BT) {
    const int id = a.top_ids[row * a.K + k];
    const bool used = id >= 0 && id < a.V;
    const float u = used ? a.top_logits[row * a.K + k] : -INFINITY;
    ids[k] = used ? id : -1;
    f[k] = u;
    mu = fmaxf(mu, u);
  }
  return mu;
}
template <typename E, int BT>
__device__ __forceinline__ void slot_sums(const DistillArgs& a, const E* z, float m, float mu, const int* ids, float* f,
                                          float (&sums)[5]) {
  sums[2] = sums[3] = sums[4] = 0.f;
  const float it = 1.f / a.tau;
  for (int k = threadIdx.x; k < a.K; k += BT) {
    const float d = (f[k] - mu) * it;  // NaN where every slot is empty or -infinity: ids[k] < 0, or f 0 below
    const float e = ids[k] < 0 || f[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(d * kLog2e);
    f[k] = e;
    if (e != 0.f) {  // a slot of no weight adds nothing, whatever its logits
      sums[2] += e;
      sums[3] = fmaf(e, d, sums[3]);
      sums[4] = fmaf(e, (to_f32<E>(z[ids[k]]) - m) * it, sums[4]);
    }
  }
}
// The columns that are not g(z) alone, over what the row's other threads wrote: the first slot of each of the
// teacher's ids writes it, and one thread the target's.
template <typename E, int BT>
__device__ __forceinline__ void slot_grads(const DistillArgs& a, E* dz, const RowGrad<E>& g, float sf, int target, float zt,
                                           const int* ids, const float* f, const float* zk) {
  const float wq = sf != 0.f ? a.alpha * a.tau * a.inv_count / sf : 0.f, w1 = (1.f - a.alpha) * a.inv_count;
  const int K = a.alpha > 0.f && sf != 0.f ? a.K : 0;  // (no teacher: none of its columns)
  for (int k = threadIdx.x; k <= K; k += BT) {
    const int id = k < K ? ids[k] : target;
    if (id < 0) continue;
    bool first = true;
    float sum = 0.f;
    for (int j = 0; j < K; j++)
      if (ids[j] == id) {
        first = first && j >= k;
        sum += f[j];
      }
    if (first) dz[id] = from_f32<E>(g(k < K ? zk[k] : zt) - (id == target ? w1 : 0.f) - wq * sum);
  }
}

// One block to a row, the row in its registers: NV 16-byte vectors a thread from the row's first
// 16-byte boundary, the elements before it and after the last whole vector one a thread.
template <typename E, int BT, int NV, bool GRAD>
__global__ __launch_bounds__(BT, 4) void k_distill_row(const DistillArgs a) {
  constexpr int VW = 16 / sizeof(E);
  __shared__ float red[2][BT / 64][8];
  extern __shared__ float slots[];  // ids[K], f[K], z of the ids[K]
  int* ids = reinterpret_cast<int*>(slots);
  float *f = slots + a.K, *zk = f + a.K;
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x, target = a.targets[row];  // (may come from host memory)
  const E* z = static_cast<const E*>(a.logits) + row * a.V;
  E* dz = static_cast<E*>(a.dlogits) + row * a.V;
  const int head = min((int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(E), a.V), nvec = (a.V - head) / VW;
  const int tail = head + nvec * VW, edge = tid < head ? tid : tail + tid - head;  // edge < V: an edge element
  const u32x4* zv = reinterpret_cast<const u32x4*>(z + head);
  u32x4* dv = reinterpret_cast<u32x4*>(dz + head);
  if (target == a.ignore) {
    if (tid == 0) a.row_loss[row] = 0.f;
    if (GRAD) {
#pragma unroll
      for (int i = 0; i < NV; i++)
        if (tid + BT * i < nvec) dv[tid + BT * i] = u32x4{0, 0, 0, 0};
      if (edge < a.V) dz[edge] = from_f32<E>(0.f);
    }
    return;
  }
  u32x4 x[NV];
#pragma unroll
  for (int i = 0; i < NV; i++) x[i] = tid + BT * i < nvec ? zv[tid + BT * i] : u32x4{0, 0, 0, 0};
  const float xe = edge < a.V ? to_f32<E>(z[edge]) : -INFINITY, zt = to_f32<E>(z[target]);
  float mx[2] = {xe, load_slots<BT>(a, row, ids, f)};
#pragma unroll
  for (int i = 0; i < NV; i++)
    if (tid + BT * i < nvec)
#pragma unroll
      for (int e = 0; e < VW; e += 2) mx[0] = max3(mx[0], element<E>(x[i], e), element<E>(x[i], e + 1));
  block_reduce<BT, 2, true>(mx, red[0]);
  const float m = mx[0];
  RowGrad<E> g{RowExp(a, m), 0.f, 0.f};
  float sums[5] = {0.f, 0.f};
  auto add = [&](float v) {
    sums[0] += g.x.soft(v);
    if (g.x.two) sums[1] += g.x.hard(v);
  };
#pragma unroll
  for (int i = 0; i < NV; i++)
    if (tid + BT * i < nvec)
#pragma unroll
      for (int e = 0; e < VW; e++) add(element<E>(x[i], e));
  if (edge < a.V) add(xe);
  slot_sums<E, BT>(a, z, m, mx[1], ids, f, sums);
  if (GRAD)
    for (int k = tid; k < a.K; k += BT) zk[k] = ids[k] < 0 ? 0.f : to_f32<E>(z[ids[k]]);
  block_reduce<BT, 5, false>(sums, red[1]);  // (and every read of the row is done)
  const float loss = row_loss(a, m, sums, zt, g);
  if (tid == 0) a.row_loss[row] = loss;
  if (!GRAD) return;
#pragma unroll
  for (int i = 0; i < NV; i++)
    if (tid + BT * i < nvec) {
      float o[VW];
#pragma unroll
      for (int e = 0; e < VW; e++) o[e] = g(element<E>(x[i], e));
      dv[tid + BT * i] = pack<E>(o);
    }
  if (edge < a.V) dz[edge] = from_f32<E>(g(xe));
  __syncthreads();
  slot_grads<E, BT>(a, dz, g, sums[2], target, zt, ids, f, zk);
}

// Any vocabulary and alignment: the row is read three times (L2), an element at a time.
template <typename E, bool GRAD>
__global__ __launch_bounds__(256) void k_distill_any(const DistillArgs a) {
  constexpr int BT = 256;
  __shared__ float red[2][BT / 64][8];
  extern __shared__ float slots[];
  int* ids = reinterpret_cast<int*>(slots);
  float *f = slots + a.K, *zk = f + a.K;
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x, target = a.targets[row];
  const E* z = static_cast<const E*>(a.logits) + row * a.V;
  E* dz = static_cast<E*>(a.dlogits) + row * a.V;
  if (target == a.ignore) {
    if (tid == 0) a.row_loss[row] = 0.f;
    if (GRAD)
      for (int v = tid; v < a.V; v += BT) dz[v] = from_f32<E>(0.f);
    return;
  }
  const float zt = to_f32<E>(z[target]);
  float mx[2] = {-INFINITY, load_slots<BT>(a, row, ids, f)};
  for (int v = tid; v < a.V; v += BT) mx[0] = fmaxf(mx[0], to_f32<E>(z[v]));
  block_reduce<BT, 2, true>(mx, red[0]);
  const float m = mx[0];
  RowGrad<E> g{RowExp(a, m), 0.f, 0.f};
  float sums[5] = {0.f, 0.f};
  for (int v = tid; v < a.V; v += BT) {
    const float x = to_f32<E>(z[v]);
    sums[0] += g.x.soft(x);
    if (g.x.two) sums[1] += g.x.hard(x);
  }
  slot_sums<E, BT>(a, z, m, mx[1], ids, f, sums);
  if (GRAD)
    for (int k = tid; k < a.K; k += BT) zk[k] = ids[k] < 0 ? 0.f : to_f32<E>(z[ids[k]]);
  block_reduce<BT, 5, false>(sums, red[1]);
  const float loss = row_loss(a, m, sums, zt, g);
  if (tid == 0) a.row_loss[row] = loss;
  if (!GRAD) return;
  for (int v = tid; v < a.V; v += BT) dz[v] = from_f32<E>(g(to_f32<E>(z[v])));
  __syncthreads();
  slot_grads<E, BT>(a, dz, g, sums[2], target, zt, ids, f, zk);
}

// sum of the row losses in double, in a fixed order: *to += it, or = it with the mark behind it (2 us of 16 rows,
// 4 of 2048; by the last block of the rows' kernel instead, counted in an atomic: no faster)
__global__ __launch_bounds__(1024) void k_distill_sum(const float* __restrict__ row_loss, int T, double* to, int add,
                                                      unsigned long long mark) {
  __shared__ double red[16];
  double s = 0;
  for (int t0 = threadIdx.x; t0 < T; t0 += 8 * 1024) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = t0 + 1024 * i < T ? row_loss[t0 + 1024 * i] : 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) s += (double)v[i];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 16; i++) s += red[i];
  if (add) {
    *to += s;
    return;
  }
  __hip_atomic_store(to, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  __builtin_amdgcn_s_waitcnt(0x0f70);  // the sum has arrived
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(to) + 1, mark, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

template <typename E, bool GRAD>
void launch(hipStream_t st, const DistillArgs& a) {
  constexpr int VW = 16 / sizeof(E);
  const dim3 grid(a.T);
  const size_t lds = (size_t)a.K * 12;
  const int vecs = a.V / VW;
  const bool same = !GRAD || ((uintptr_t)a.logits & 15) == ((uintptr_t)a.dlogits & 15);
#define ROW(bt, nv) hipLaunchKernelGGL((k_distill_row<E, bt, nv, GRAD>), grid, dim3(bt), lds, st, a)
  if (!same || a.T >= 1 << 22 || vecs > 1024 * 13)
    hipLaunchKernelGGL((k_distill_any<E, GRAD>), grid, dim3(256), lds, st, a);
  else if (vecs <= 256)
    ROW(256, 1);
  else if (vecs <= 256 * 4)
    ROW(256, 4);
  else if (vecs <= 256 * 8)
    ROW(256, 8);
  else if (vecs <= 256 * 16)
    ROW(256, 16);
  else if (vecs <= 512 * 16)
    ROW(512, 16);
  else
    ROW(1024, 13);
#undef ROW
}

}  // namespace

hipError_t launch_distill(hipStream_t st, const DistillArgs& a, bool bf16, double* sum, bool add, unsigned long long mark) {
  if (a.T <= 0 || a.T >= 1 << 24 || a.V <= 0 || a.K <= 0 || a.K > kDistillTop || !a.logits || !a.targets || !a.top_ids ||
      !a.top_logits || !a.row_loss || !sum)
    return hipErrorInvalidValue;
  if (bf16)
    a.dlogits ? launch<bf16_t, true>(st, a) : launch<bf16_t, false>(st, a);
  else
    a.dlogits ? launch<float, true>(st, a) : launch<float, false>(st, a);
  hipLaunchKernelGGL(k_distill_sum, dim3(1), dim3(1024), 0, st, a.row_loss, a.T, sum, add ? 1 : 0, mark);
  return hipGetLastError();
}

}  // namespace fh
