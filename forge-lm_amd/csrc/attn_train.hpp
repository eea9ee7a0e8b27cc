// attn_train.hpp -- causal attention of the op-level backend: what its forward (attn_train.hip)
// and backward (attn_train_bwd.hip) kernels share.
//
// A wave owns 32 rows of one axis (queries, or keys) and walks the other axis in LDS tiles.  With
// v_mfma_f32_32x32x* two products cover everything, and neither moves a score between lanes:
//   rows  acc[r][i] += sum_d tile[r][d] own[i][d]   scores: lane l holds own row l % 32 and, in
//                                                   register r, tile row (r/4)*8 + (l/32)*4 + r%4
//   cols  acc[d][i] += sum_r tile[r][d] w[r][i]     the score registers are the B operand as they
//                                                   are; the tile is read transposed
// fp32 tensors multiply on v_mfma_f32_32x32x2_f32 (exact fp32 products and sums), bf16 ones on
// v_mfma_f32_32x32x16_bf16 with fp32 sums; softmax statistics and sums are fp32 in both.
#pragma once

#include "kernels.hpp"

#include <type_traits>

namespace fh {

typedef __bf16 at_bf16x8 __attribute__((ext_vector_type(8)));
typedef float at_f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int at_u32x4 __attribute__((ext_vector_type(4)));
typedef short at_s16x4 __attribute__((ext_vector_type(4)));

template <int I>
constexpr std::integral_constant<int, I> at_int{};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

constexpr __device__ __forceinline__ int at_row0(int r) { return (r >> 2) * 8 + (r & 3); }  // of the lower lanes
__device__ __forceinline__ int at_row(int lane, int r) { return at_row0(r) + (lane >> 5) * 4; }

__device__ __forceinline__ void at_zero(at_f32x16& v) {
#pragma unroll
  for (int r = 0; r < 16; r++) v[r] = 0.f;
}

// Rows of a strided matrix: `rows` of them from base, hd elements each, `stride` apart.  Elements
// past either end read as zeros.  VEC: base, stride and hd are multiples of 16 bytes.
template <typename E>
struct AtRows {
  __amdgpu_buffer_rsrc_t rsrc;
  int stride, hd;  // bytes, elements
};
template <typename E>
__device__ __forceinline__ AtRows<E> at_rows(const E* base, int rows, int stride, int hd) {
  const int n = rows > 0 ? ((rows - 1) * stride + hd) * (int)sizeof(E) : 0;
  return {__builtin_amdgcn_make_buffer_rsrc(const_cast<E*>(base), (short)0, n, 0x00020000), stride * (int)sizeof(E), hd};
}
template <typename E, bool VEC>
__device__ __forceinline__ at_u32x4 at_chunk(const AtRows<E>& m, int row, int chunk) {
  constexpr int CE = 16 / sizeof(E);
  constexpr int kPast = 0x7ffffff0;  // past every resource (at most 2^30 bytes)
  if constexpr (VEC) {
    return __builtin_amdgcn_raw_buffer_load_b128(m.rsrc, chunk * CE < m.hd ? row * m.stride + chunk * 16 : kPast, 0, 0);
  } else {
    at_u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < CE; e++) {
      const int at = chunk * CE + e < m.hd ? row * m.stride + (chunk * CE + e) * (int)sizeof(E) : kPast;
      if constexpr (sizeof(E) == 2)
        v[e / 2] |= (unsigned)__builtin_amdgcn_raw_buffer_load_b16(m.rsrc, at, 0, 0) << (16 * (e & 1));
      else
        v[e] = __builtin_amdgcn_raw_buffer_load_b32(m.rsrc, at, 0, 0);
    }
    return v;
  }
}

// The two products and the operand layouts of a type, for heads padded to HD.
template <typename E, int HD>
struct AtMma;

template <int HD>
struct AtMma<__bf16, HD> {
  typedef __bf16 E;
  static constexpr int kChunks = HD / 8;  // 16-byte chunks of a row
  static constexpr int kStride = HD;      // LDS elements of a row
  // Chunks of a row are permuted so that the 16 lanes of a 16-byte read (16 rows, one chunk) and the
  // 32 of a transposing read (4 rows, 64 bytes of each) fall on distinct banks.
  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (HD == 32) return (row >> 2) & 3;
    if constexpr (HD == 64) return ((row & 2) << 1) | ((row & 4) >> 1) | ((row >> 3) & 1);
    return ((row & 3) << 2) | ((row & 4) >> 1) | ((row >> 3) & 1);
  }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * kStride + 8 * (chunk ^ swizzle(row)); }
  struct Own {
    at_bf16x8 v[HD / 16];  // own row l % 32, dims 16 kk + 8 (l / 32) ..
  };
  template <bool VEC>
  static __device__ __forceinline__ Own own(const AtRows<E>& m, int row, int lane) {
    Own o;
#pragma unroll
    for (int kk = 0; kk < HD / 16; kk++)
      o.v[kk] = __builtin_bit_cast(at_bf16x8, at_chunk<E, VEC>(m, row, 2 * kk + (lane >> 5)));
    return o;
  }
  // a lane's half of the dot product of two own rows
  static __device__ __forceinline__ float dot(const Own& a, const Own& b) {
    float s = 0.f;
#pragma unroll
    for (int kk = 0; kk < HD / 16; kk++)
#pragma unroll
      for (int e = 0; e < 8; e++) s = fmaf((float)a.v[kk][e], (float)b.v[kk][e], s);
    return s;
  }
  // 32 rows of a tile as the operand of `rows`
  struct Rows {
    at_bf16x8 v[HD / 16];
  };
  static __device__ __forceinline__ Rows load_rows(const E* tile, int row0, int lane) {
    Rows f;
#pragma unroll
    for (int kk = 0; kk < HD / 16; kk++)
      f.v[kk] = *reinterpret_cast<const at_bf16x8*>(tile + at(row0 + (lane & 31), 2 * kk + (lane >> 5)));
    return f;
  }
  static __device__ __forceinline__ void rows(at_f32x16& acc, const Rows& f, const Own& o) {
#pragma unroll
    for (int kk = 0; kk < HD / 16; kk++) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.v[kk], o.v[kk], acc, 0, 0, 0);
  }
  // 32 rows of a tile as the operand of `cols`: a transposing read takes 4 rows x 16 dims per 16 lanes; lane
  // i points at 4 dims of row i / 4 and gets dim i of the 4 rows
  struct Cols {
    union {
      at_s16x4 h[2];
      at_bf16x8 v;
    } f[2][HD / 32];
  };
  static __device__ __forceinline__ Cols load_cols(const E* tile, int row0, int lane) {
    Cols c;
#pragma unroll
    for (int kk = 0; kk < 2; kk++)
#pragma unroll
      for (int dt = 0; dt < HD / 32; dt++) {
        const int row = row0 + 16 * kk + 4 * (lane >> 5) + ((lane >> 2) & 3);
        const int dim = dt * 32 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
        for (int j = 0; j < 2; j++)
          c.f[kk][dt].h[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) at_s16x4*)(tile + at(row + 8 * j, dim >> 3) + (dim & 7)));
      }
    return c;
  }
  // w is rounded to bf16: the probabilities (or their gradients) enter a product as the tensors do
  static __device__ __forceinline__ void cols(at_f32x16 (&acc)[HD / 32], const Cols& c, const at_f32x16& w, int) {
#pragma unroll
    for (int kk = 0; kk < 2; kk++) {
      at_bf16x8 b;
#pragma unroll
      for (int e = 0; e < 8; e++) b[e] = (__bf16)w[8 * kk + e];
#pragma unroll
      for (int dt = 0; dt < HD / 32; dt++)
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(c.f[kk][dt].v, b, acc[dt], 0, 0, 0);
    }
  }
};

template <int HD>
struct AtMma<float, HD> {
  typedef float E;
  static constexpr int kChunks = HD / 4;
  static constexpr int kStride = HD;
  // 16 rows of one chunk on distinct banks; the 32 lanes of a column read share a row
  static __device__ __forceinline__ int swizzle(int row) { return HD == 32 ? (row >> 1) & 7 : row & 15; }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * kStride + 4 * (chunk ^ swizzle(row)); }
  struct Own {
    float v[HD / 2];  // own row l % 32, dims (l / 32) HD / 2 ..: a product step pairs dims d and d + HD / 2
  };
  template <bool VEC>
  static __device__ __forceinline__ Own own(const AtRows<E>& m, int row, int lane) {
    Own o;
#pragma unroll
    for (int c = 0; c < HD / 8; c++) {
      const at_u32x4 x = at_chunk<E, VEC>(m, row, (lane >> 5) * (HD / 8) + c);
#pragma unroll
      for (int e = 0; e < 4; e++) o.v[4 * c + e] = __uint_as_float(x[e]);
    }
    return o;
  }
  static __device__ __forceinline__ float dot(const Own& a, const Own& b) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 2; i++) s = fmaf(a.v[i], b.v[i], s);
    return s;
  }
  // (an MFMA takes 64 cycles here and one or two LDS reads: they are read where they are used)
  struct Rows {
    const E* tile;
    int row, half;
  };
  static __device__ __forceinline__ Rows load_rows(const E* tile, int row0, int lane) {
    return {tile, row0 + (lane & 31), lane >> 5};
  }
  static __device__ __forceinline__ void rows(at_f32x16& acc, const Rows& f, const Own& o) {
#pragma unroll
    for (int c = 0; c < HD / 8; c++) {
      const float4 a = *reinterpret_cast<const float4*>(f.tile + at(f.row, f.half * (HD / 8) + c));
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, o.v[4 * c], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, o.v[4 * c + 1], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, o.v[4 * c + 2], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, o.v[4 * c + 3], acc, 0, 0, 0);
    }
  }
  struct Cols {
    const E* tile;
  };
  static __device__ __forceinline__ Cols load_cols(const E* tile, int row0, int) { return {tile + row0 * kStride}; }
  // the tile's rows start at a multiple of 32: of a row's swizzle, bits 2 (HD 32) or 3 (`high`) and up are
  // constants
  static __device__ __forceinline__ void cols(at_f32x16 (&acc)[HD / 32], const Cols& f, const at_f32x16& w, int lane) {
    const int half = lane >> 5, c = (lane & 31) >> 2;
    const E* t = f.tile + 4 * half * kStride + (lane & 3);
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int row = (r >> 2) * 8 + (r & 3), high = (r >> 2) & 1;
      const int low = HD == 32 ? (c ^ (2 * half + ((r & 3) >> 1))) ^ (4 * high) : c ^ (4 * half + (r & 3));
#pragma unroll
      for (int dt = 0; dt < HD / 32; dt++)
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(t[row * kStride + 4 * low + (HD == 32 ? 0 : 32 * (dt ^ high))], w[r],
                                                       acc[dt], 0, 0, 0);
    }
  }
};

// SR rows of m into an LDS tile, by the block's 256 threads.
template <typename E, int HD, int SR, bool VEC>
__device__ __forceinline__ void at_stage(E* tile, const AtRows<E>& m, int tid) {
  typedef AtMma<E, HD> M;
#pragma unroll
  for (int i = 0; i < SR * M::kChunks / 256; i++) {
    const int row = (tid + 256 * i) / M::kChunks, c = (tid + 256 * i) % M::kChunks;
    *reinterpret_cast<at_u32x4*>(tile + M::at(row, c)) = at_chunk<E, VEC>(m, row, c);
  }
}

// ROWS rows of m straight into an LDS tile: 1 KB pieces (64 lanes x 16 bytes, contiguous in LDS),
// every WAVES-th of them from `first` by this wave.  A lane asks for the chunk whose place is its own.
// Chunks past either end of m arrive as zeros.
template <typename E, int HD, int ROWS, int WAVES>
__device__ __forceinline__ void at_fetch(E* tile, const AtRows<E>& m, int first, int lane) {
  typedef AtMma<E, HD> M;
  constexpr int CE = 16 / sizeof(E), RP = 64 / M::kChunks, N = ROWS / RP / WAVES;
  static_assert(N * RP * WAVES == ROWS, "pieces");
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int row0 = (first + WAVES * i) * RP, row = row0 + lane / M::kChunks;
    const int c = (lane % M::kChunks) ^ M::swizzle(row);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(m.rsrc, (__attribute__((address_space(3))) void*)(tile + row0 * M::kStride), 16,
                                             c * CE < m.hd ? row * m.stride + c * 16 : 0x7ffffff0, 0, 0, 0);
  }
}

// Waits until at most VM of this wave's requests are on their way (and, VM < 0, no count is asked for) and
// its LDS reads are done.  (The builtin, unlike a wait in inline assembly, also tells the compiler so.)
template <int VM>
__device__ __forceinline__ void at_wait() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  constexpr int vm = VM < 0 || VM > 63 ? 63 : VM;
  __builtin_amdgcn_s_waitcnt(0x0070 | (vm & 15) | (vm >> 4) << 14);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
// Every wave's requests have landed and every wave's LDS reads are done.
__device__ __forceinline__ void at_landed() {
  at_wait<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// acc^T (dims x own rows) times f to the 32 rows from `base` on (stride elements apart, hd of them each), of
// which `rows` exist and the first `len` count: the others are zeros.  LDS: by whole 16-byte chunks of a
// row through the wave's part of LDS, `tile` of 32 HD elements; the pieces that a lane holds (4 dims of
// 32 different rows) would be partial writes of every line (dk and dv of 8 x 1024 rows: 42 us, 35 without
// the stores).
template <typename E, int HD, bool VEC, bool LDS>
__device__ __forceinline__ void at_store(E* base, int stride, const at_f32x16 (&acc)[HD / 32], float f, int rows, int len,
                                         int hd, E* tile, int lane) {
  typedef AtMma<E, HD> M;
  typedef E e4 __attribute__((ext_vector_type(4)));
  constexpr int CE = 16 / sizeof(E);
  const int i = lane & 31;
#pragma unroll
  for (int dt = 0; dt < HD / 32; dt++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int dim = dt * 32 + 8 * g + 4 * (lane >> 5);
      e4 v = {(E)(acc[dt][4 * g] * f), (E)(acc[dt][4 * g + 1] * f), (E)(acc[dt][4 * g + 2] * f),
              (E)(acc[dt][4 * g + 3] * f)};
      if (i >= len) v = e4{(E)0.f, (E)0.f, (E)0.f, (E)0.f};
      if constexpr (LDS) {
        *reinterpret_cast<e4*>(tile + M::at(i, dim / CE) + dim % CE) = v;
      } else if constexpr (VEC) {
        if (i < rows && dim < hd) *reinterpret_cast<e4*>(base + (size_t)i * stride + dim) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (i < rows && dim + e < hd) base[(size_t)i * stride + dim + e] = v[e];
      }
    }
  if constexpr (LDS) {
    constexpr int RP = 64 / M::kChunks;
#pragma unroll
    for (int p = 0; p < 32 / RP; p++) {
      const int row = p * RP + lane / M::kChunks, c = lane % M::kChunks;
      const at_u32x4 v = *reinterpret_cast<const at_u32x4*>(tile + M::at(row, c));
      if (row < rows && c * CE < hd) *reinterpret_cast<at_u32x4*>(base + (size_t)row * stride + c * CE) = v;
    }
  }
}

// How a block goes through the axis it walks.
// KS == 1: its four waves own 32 rows each of the other axis and share tiles of kRows rows, which are
// requested one ahead into the other of two buffers (at_walk).
// KS == 4: they own the same 32 rows; each takes every fourth 32-row part through tiles of its own,
// without a barrier, and the sums are joined at the end.  A part's two tiles have one place each: the
// next part's is requested as soon as a tile has been read for the last time, while the products with
// the other one run, so that two blocks fit a CU.
template <typename E, int HD, int KS, bool VEC>
struct AtPlan {
  static constexpr int kOwn = 128 / KS;  // rows of a block
  static constexpr int kRows = KS == 4 ? 32 : sizeof(E) == 4 && HD == 128 ? 32 : 64;
  static constexpr int kParts = kRows / 32;   // 32-row parts of a tile
  static constexpr int kTile = kRows * HD;    // elements of one operand's tile
  static constexpr int kLoads = kTile * (int)sizeof(E) / 1024 / (KS == 4 ? 1 : 4);  // a wave's requests for a tile
  static constexpr int kBufs = VEC && KS == 1 ? 2 : 1;
  static constexpr int kBytes = 2 * kTile * KS * (int)sizeof(E);  // a buffer: both operands, all waves
  static constexpr bool kStaged = VEC && KS == 1 && 128 * HD * (int)sizeof(E) <= kBytes;  // at_store's LDS fits one
};

// A tile of the operand x: by all four waves of the block (KS == 1), or by this wave alone.
template <typename E, int HD, int KS, bool VEC>
__device__ __forceinline__ void at_load(E* tile, const AtRows<E>& x, int w, int lane) {
  typedef AtPlan<E, HD, KS, VEC> P;
  static_assert(VEC || KS == 1, "element loads are shared by the block");
  if constexpr (VEC)
    at_fetch<E, HD, P::kRows, KS == 4 ? 1 : 4>(tile, x, KS == 4 ? 0 : w, lane);
  else
    at_stage<E, HD, P::kRows, false>(tile, x, 64 * w + lane);
}
// KS == 1: the steps 0 .. n - 1 of a walk: step kt computes on a buffer whose tiles have landed while those of
// kt + 1 are on their way to the other.  The two buffers are LDS variables of their own and appear by
// name in code of their own, so that the compiler does not make the reads of one wait for the other.
template <typename P, typename F, typename C>
__device__ __forceinline__ void at_walk(int n, char* even, char* odd, const F& fetch, const C& compute) {
  if constexpr (P::kBufs == 2) {
    fetch(0, even);
    for (int kt = 0; kt < n; kt += 2) {
      at_landed();
      if (kt + 1 < n) fetch(kt + 1, odd);
      compute(kt, even);
      if (kt + 1 == n) break;
      at_landed();
      if (kt + 2 < n) fetch(kt + 2, even);
      compute(kt + 1, odd);
    }
  } else {
    for (int kt = 0; kt < n; kt++) {
      at_landed();  // the last tile's reads are done
      fetch(kt, even);
      at_landed();
      compute(kt, even);
    }
  }
}

// Block -> (block of the axis, group = sequence * heads + head) of a causal launch over nblk * G
// blocks; block 0 of the axis is the one with the most work, and is started first.  Workgroups reach
// the 8 XCDs round-robin.  Sequences of one length: when 8 divides G, an XCD takes whole neighbouring
// groups, so that what their blocks share is fetched into its L2 only; every other 32 of its blocks (one for
// each of its CUs) come in reverse, so that a CU's blocks add up to the same (dq of 8 x 1024 rows, three
// blocks to a CU: 32.1 -> 30.5 us).  Sequences of their own lengths:
// a group's blocks go to all XCDs in turn, which evens out what long ones cost (4 x up to 1333 rows, 16
// heads of 128, dq: 60 us with groups kept together, an XCD idle for half of it).
struct AtBlock {
  int blk, g;
};
__device__ __forceinline__ AtBlock at_block(int L, int G, int ragged) {
  if (!ragged && G % 8 == 0) {
    const int gx = G / 8, i = L >> 3, first = i & ~31, n = min(32, (int)(gridDim.x >> 3) - first);
    const int s = i & 32 ? first + n - 1 - (i - first) : i;
    return {s / gx, (L & 7) * gx + s % gx};
  }
  const int blk = L / G, i = L % G;
  return {blk, ragged && G % 2 == 0 ? (i + blk) % G : i};
}

__device__ __forceinline__ int at_len(const AttnTrain& a, int b) {
  if (!a.ragged) return a.T;
  return __builtin_amdgcn_readfirstlane(a.lens_dev ? a.lens_dev[b] : a.lens[b]);
}

}  // namespace fh
