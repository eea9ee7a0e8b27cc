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

template <typename E>
__device__ __forceinline__ float element(const u32x4& v, int e);
template <>
__device__ __forceinline__ float element<float>(const u32x4& v, int e) { return __uint_as_float(v[e]); }
template <>
__device__ __forceinline__ float element<bf16_t>(const u32x4& v, int e) {
  return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
}
template <typename E>
__device__ __forceinline__ void put(u32x4& v, int e, float f);
template <>
__device__ __forceinline__ void put<float>(u32x4& v, int e, float f) { v[e] = __float_as_uint(f); }
template <>
__device__ __forceinline__ void put<bf16_t>(u32x4& v, int e, float f) {
  v[e >> 1] = e & 1 ? v[e >> 1] | (unsigned)bf16_rn(f) << 16 : (unsigned)bf16_rn(f);
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

// What a row's columns need once its sums are known: g(z) = at 2^((z - m) ct) + a1 2^((z - m) c1).
struct RowGrad {
  float m, ct, at, c1, a1;
  bool two;
  __device__ __forceinline__ float operator()(float z) const {
    const float d = z - m;
    float g = at * __builtin_amdgcn_exp2f(d * ct);
    if (two) g = fmaf(a1, __builtin_amdgcn_exp2f(d * c1), g);
    return g;
  }
};

// The row's loss and gradient weights from its sums.  sums: 2^((z - m) ct), 2^((z - m) c1) (the same
// where one exponential serves both), f, f u', f z'.
__device__ __forceinline__ float row_loss(const DistillArgs& a, float m, const float (&sums)[5], float zt, bool two,
                                          RowGrad& g) {
  const float st = sums[0], s1 = two ? sums[1] : sums[0], sf = sums[2];
  const bool kept = sf > 0.f || sf != sf;  // a row with a used slot (a NaN among them goes on)
  float loss = 0.f;
  if (a.alpha > 0.f && kept)
    loss = a.alpha * a.tau * a.tau *
           ((sums[3] - sums[4]) / sf + (__builtin_amdgcn_logf(st) - __builtin_amdgcn_logf(sf)) * kLn2);
  if (a.alpha < 1.f) loss += (1.f - a.alpha) * (__builtin_amdgcn_logf(s1) * kLn2 - (zt - m));
  const float wt = kept ? a.alpha * a.tau * a.inv_count : 0.f, w1 = (1.f - a.alpha) * a.inv_count;
  g.m = m;
  g.two = two;
  g.c1 = kLog2e;
  g.a1 = w1 / s1;
  if (two) {
    g.ct = kLog2e / a.tau;
    g.at = wt / st;
  } else {  // tau 1, or one of the two terms alone
    g.ct = a.alpha > 0.f ? kLog2e / a.tau : kLog2e;
    g.at = (wt + w1) / st;
    g.a1 = 0.f;
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
// The columns that the teacher touches: the first slot of each id writes it.
template <typename E, int BT>
__device__ __forceinline__ void slot_grads(const DistillArgs& a, const E* z, E* dz, const RowGrad& g, float sf, int target,
                                           const int* ids, const float* f, const float* zk) {
  const float wq = a.alpha * a.tau * a.inv_count / sf, w1 = (1.f - a.alpha) * a.inv_count;
  for (int k = threadIdx.x; k < a.K; k += BT) {
    const int id = ids[k];
    if (id < 0) continue;
    bool first = true;
    float sum = 0.f;
    for (int j = 0; j < a.K; j++)
      if (ids[j] == id) {
        first = first && j >= k;
        sum += f[j];
      }
    if (first) dz[id] = from_f32<E>(g(zk[k]) - (id == target ? w1 : 0.f) - wq * sum);
  }
}

// One block to a row, the row in its registers: NV 16-byte vectors a thread from the row's first
// 16-byte boundary, the elements before it and after the last whole vector one a thread.
template <typename E, int BT, int NV, bool GRAD>
__global__ __launch_bounds__(BT) void k_distill_row(const DistillArgs a) {
  constexpr int VW = 16 / sizeof(E);
  __shared__ float red[2][BT / 64][8];
  extern __shared__ float slots[];  // ids[K], f[K], z of the ids[K]
  int* ids = reinterpret_cast<int*>(slots);
  float *f = slots + a.K, *zk = f + a.K;
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x, target = a.targets[row];
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
      for (int e = 0; e < VW; e++) mx[0] = fmaxf(mx[0], element<E>(x[i], e));
  block_reduce<BT, 2, true>(mx, red[0]);
  const float m = mx[0];
  const bool two = a.alpha > 0.f && a.alpha < 1.f && a.tau != 1.f;
  const float ct = a.alpha > 0.f ? kLog2e / a.tau : kLog2e;
  float sums[5] = {0.f, 0.f};
  auto add = [&](float v) {
    sums[0] += __builtin_amdgcn_exp2f((v - m) * ct);
    if (two) sums[1] += __builtin_amdgcn_exp2f((v - m) * kLog2e);
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
  RowGrad g;
  const float loss = row_loss(a, m, sums, zt, two, g);
  if (tid == 0) a.row_loss[row] = loss;
  if (!GRAD) return;
  const float w1 = (1.f - a.alpha) * a.inv_count;
#pragma unroll
  for (int i = 0; i < NV; i++)
    if (tid + BT * i < nvec) {
      u32x4 o;
#pragma unroll
      for (int e = 0; e < VW; e++) {
        float v = g(element<E>(x[i], e));
        if (head + (tid + BT * i) * VW + e == target) v -= w1;
        put<E>(o, e, v);
      }
      dv[tid + BT * i] = o;
    }
  if (edge < a.V) dz[edge] = from_f32<E>(g(xe) - (edge == target ? w1 : 0.f));
  if (a.alpha == 0.f || sums[2] == 0.f) return;  // no teacher: none of its columns
  __syncthreads();
  slot_grads<E, BT>(a, z, dz, g, sums[2], target, ids, f, zk);
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
  const bool two = a.alpha > 0.f && a.alpha < 1.f && a.tau != 1.f;
  const float ct = a.alpha > 0.f ? kLog2e / a.tau : kLog2e;
  float sums[5] = {0.f, 0.f};
  for (int v = tid; v < a.V; v += BT) {
    const float d = to_f32<E>(z[v]) - m;
    sums[0] += __builtin_amdgcn_exp2f(d * ct);
    if (two) sums[1] += __builtin_amdgcn_exp2f(d * kLog2e);
  }
  slot_sums<E, BT>(a, z, m, mx[1], ids, f, sums);
  if (GRAD)
    for (int k = tid; k < a.K; k += BT) zk[k] = ids[k] < 0 ? 0.f : to_f32<E>(z[ids[k]]);
  block_reduce<BT, 5, false>(sums, red[1]);
  RowGrad g;
  const float loss = row_loss(a, m, sums, zt, two, g);
  if (tid == 0) a.row_loss[row] = loss;
  if (!GRAD) return;
  const float w1 = (1.f - a.alpha) * a.inv_count;
  for (int v = tid; v < a.V; v += BT) dz[v] = from_f32<E>(g(to_f32<E>(z[v])) - (v == target ? w1 : 0.f));
  if (a.alpha == 0.f || sums[2] == 0.f) return;  // no teacher: none of its columns
  __syncthreads();
  slot_grads<E, BT>(a, z, dz, g, sums[2], target, ids, f, zk);
}

// sum of the row losses in double, in a fixed order: acc[0] += it, or acc[1] = it
__global__ __launch_bounds__(1024) void k_distill_sum(const float* __restrict__ row_loss, int T, double* acc, int add) {
  __shared__ double red[16];
  double s = 0;
  for (int t = threadIdx.x; t < T; t += 1024) s += (double)row_loss[t];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 16; i++) s += red[i];
  if (add)
    acc[0] += s;
  else
    acc[1] = s;
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
  else if (vecs <= 1024)
    ROW(1024, 1);
  else if (vecs <= 1024 * 2)
    ROW(1024, 2);
  else if (vecs <= 1024 * 4)
    ROW(1024, 4);
  else if (vecs <= 1024 * 8)
    ROW(1024, 8);
  else
    ROW(1024, 13);
#undef ROW
}

}  // namespace

hipError_t launch_distill(hipStream_t st, const DistillArgs& a, bool bf16, double* acc, bool add) {
  if (a.T <= 0 || a.T >= 1 << 24 || a.V <= 0 || a.K <= 0 || a.K > kDistillTop || !a.logits || !a.targets || !a.top_ids ||
      !a.top_logits || !a.row_loss || !acc)
    return hipErrorInvalidValue;
  if (bf16)
    a.dlogits ? launch<bf16_t, true>(st, a) : launch<bf16_t, false>(st, a);
  else
    a.dlogits ? launch<float, true>(st, a) : launch<float, false>(st, a);
  hipLaunchKernelGGL(k_distill_sum, dim3(1), dim3(1024), 0, st, a.row_loss, a.T, acc, add ? 1 : 0);
  return hipGetLastError();
}

}  // namespace fh
