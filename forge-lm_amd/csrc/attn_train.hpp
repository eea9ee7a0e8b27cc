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

namespace fh {

typedef __bf16 at_bf16x8 __attribute__((ext_vector_type(8)));
typedef float at_f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int at_u32x4 __attribute__((ext_vector_type(4)));
typedef short at_s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ int at_row(int lane, int r) { return (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3); }

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
  static __device__ __forceinline__ void rows(at_f32x16& acc, const E* tile, int row0, const Own& o, int lane) {
    const int row = row0 + (lane & 31);
#pragma unroll
    for (int kk = 0; kk < HD / 16; kk++)
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          *reinterpret_cast<const at_bf16x8*>(tile + at(row, 2 * kk + (lane >> 5))), o.v[kk], acc, 0, 0, 0);
  }
  // w is rounded to bf16: the probabilities (or their gradients) enter a product as the tensors do
  static __device__ __forceinline__ void cols(at_f32x16 (&acc)[HD / 32], const E* tile, int row0, const at_f32x16& w,
                                              int lane) {
#pragma unroll
    for (int kk = 0; kk < 2; kk++) {
      at_bf16x8 b;
#pragma unroll
      for (int e = 0; e < 8; e++) b[e] = (__bf16)w[8 * kk + e];
      // a transposing read takes 4 rows x 16 dims per 16 lanes: lane i points at 4 dims of row i / 4 and
      // gets dim i of the 4 rows
      const int row = row0 + 16 * kk + 4 * (lane >> 5) + ((lane >> 2) & 3);
#pragma unroll
      for (int dt = 0; dt < HD / 32; dt++) {
        const int dim = dt * 32 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        union {
          at_s16x4 h[2];
          at_bf16x8 v;
        } a;
#pragma unroll
        for (int j = 0; j < 2; j++)
          a.h[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) at_s16x4*)(tile + at(row + 8 * j, dim >> 3) + (dim & 7)));
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b, acc[dt], 0, 0, 0);
      }
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
  static __device__ __forceinline__ void rows(at_f32x16& acc, const E* tile, int row0, const Own& o, int lane) {
    const int row = row0 + (lane & 31);
#pragma unroll
    for (int c = 0; c < HD / 8; c++) {
      const float4 a = *reinterpret_cast<const float4*>(tile + at(row, (lane >> 5) * (HD / 8) + c));
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, o.v[4 * c], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, o.v[4 * c + 1], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, o.v[4 * c + 2], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, o.v[4 * c + 3], acc, 0, 0, 0);
    }
  }
  // row0 a multiple of 32: of a row's swizzle, bits 2 (HD 32) or 3 (`high`) and up are constants
  static __device__ __forceinline__ void cols(at_f32x16 (&acc)[HD / 32], const E* tile, int row0, const at_f32x16& w,
                                              int lane) {
    const int half = lane >> 5, c = (lane & 31) >> 2;
    const E* t = tile + (row0 + 4 * half) * kStride + (lane & 3);
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

// This wave's requests have landed and its LDS reads are done; BLOCK: every wave's of the block.  (The
// builtin, unlike a wait in inline assembly, also tells the compiler that nothing is in flight.)
template <bool BLOCK>
__device__ __forceinline__ void at_landed() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
  if constexpr (BLOCK) __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// acc^T (dims x own rows) times f to row `row` (a pointer to its hd elements) of the lane's own row
template <typename E, int HD, bool VEC>
__device__ __forceinline__ void at_store(E* row, const at_f32x16 (&acc)[HD / 32], float f, int hd, int lane) {
  typedef E e4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int dt = 0; dt < HD / 32; dt++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int dim = dt * 32 + 8 * g + 4 * (lane >> 5);
      const e4 v = {(E)(acc[dt][4 * g] * f), (E)(acc[dt][4 * g + 1] * f), (E)(acc[dt][4 * g + 2] * f),
                    (E)(acc[dt][4 * g + 3] * f)};
      if constexpr (VEC) {
        if (dim < hd) *reinterpret_cast<e4*>(row + dim) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (dim + e < hd) row[dim + e] = v[e];
      }
    }
}

// How a block goes through the axis it walks.  KS == 1: its four waves own 32 rows each of the other
// axis and share tiles of kRows rows.  KS == 4: they own the same 32 rows and each walks every fourth
// 32-row part through tiles of its own, without a barrier; their sums are joined at the end.
// Tiles are requested one ahead into the other of two buffers (one buffer where two do not fit).
template <typename E, int HD, int KS, bool VEC>
struct AtPlan {
  static constexpr int kOwn = 128 / KS;  // rows of a block
  static constexpr int kRows = KS == 4 ? 128 : sizeof(E) == 4 && HD == 128 ? 32 : 64;
  static constexpr int kParts = kRows / (32 * KS);     // 32-row parts of a wave
  static constexpr int kTile = (KS == 4 ? 32 : kRows) * HD;  // elements of one operand's tile
  static constexpr int kBufs = VEC && !(KS == 4 && sizeof(E) == 4 && HD == 128) ? 2 : 1;
  static constexpr int kBytes = 2 * kTile * KS * (int)sizeof(E);  // a buffer: both operands, all waves
};

// The tiles of two operands into `tiles` (the second kTile elements on): by all four waves of the
// block (KS == 1), or by this wave alone.
template <typename E, int HD, int KS, bool VEC>
__device__ __forceinline__ void at_load(E* tiles, const AtRows<E>& x, const AtRows<E>& y, int w, int lane) {
  typedef AtPlan<E, HD, KS, VEC> P;
  if constexpr (VEC) {
    constexpr int ROWS = KS == 4 ? 32 : P::kRows, WAVES = KS == 4 ? 1 : 4;
    at_fetch<E, HD, ROWS, WAVES>(tiles, x, KS == 4 ? 0 : w, lane);
    at_fetch<E, HD, ROWS, WAVES>(tiles + P::kTile, y, KS == 4 ? 0 : w, lane);
  } else {
    static_assert(KS == 1, "element loads are shared by the block");
    at_stage<E, HD, P::kRows, false>(tiles, x, 64 * w + lane);
    at_stage<E, HD, P::kRows, false>(tiles + P::kTile, y, 64 * w + lane);
  }
}
// The steps 0 .. n - 1 of a walk: step kt computes on a buffer whose tiles have landed while those of
// kt + 1 are on their way to the other.  The two buffers are LDS variables of their own and appear by
// name in code of their own, so that the compiler does not make the reads of one wait for the other.
template <typename P, int KS, typename F, typename C>
__device__ __forceinline__ void at_walk(int n, char* even, char* odd, const F& fetch, const C& compute) {
  if constexpr (P::kBufs == 2) {
    fetch(0, even);
    for (int kt = 0; kt < n; kt += 2) {
      at_landed<KS == 1>();
      if (kt + 1 < n) fetch(kt + 1, odd);
      compute(kt, even);
      if (kt + 1 == n) break;
      at_landed<KS == 1>();
      if (kt + 2 < n) fetch(kt + 2, even);
      compute(kt + 1, odd);
    }
  } else {
    for (int kt = 0; kt < n; kt++) {
      at_landed<KS == 1>();  // the last tile's reads are done
      fetch(kt, even);
      at_landed<KS == 1>();
      compute(kt, even);
    }
  }
}

// Block -> (block of the axis, group = sequence * heads + head) of a causal launch over nblk * G
// blocks; block 0 of the axis is the one with the most work, and is started first.  Workgroups reach
// the 8 XCDs round-robin: when 8 divides G, an XCD takes whole neighbouring groups, so that what their
// blocks share is fetched into its L2 only.
struct AtBlock {
  int blk, g;
};
__device__ __forceinline__ AtBlock at_block(int L, int G) {
  if (G % 8 == 0) {
    const int s = L >> 3, gx = G / 8;
    return {s / gx, (L & 7) * gx + s % gx};
  }
  return {L / G, L % G};
}

__device__ __forceinline__ int at_len(const AttnTrain& a, int b) {
  if (!a.ragged) return a.T;
  return __builtin_amdgcn_readfirstlane(a.lens_dev ? a.lens_dev[b] : a.lens[b]);
}

}  // namespace fh
