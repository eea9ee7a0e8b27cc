// attn_train.hpp -- causal attention of the op-level backend: what its forward (attn_train.hip)
// and backward (attn_train_bwd.hip) kernels share.
//
// A wave owns 32 rows of one axis (queries, or keys) and walks the other axis in LDS tiles.  With
// v_mfma_f32_32x32x* two products cover everything, and neither moves a score between lanes:
//   rows  acc[r][i] += sum_d tile[r][d] own[i][d]   scores: lane l holds own row l % 32 and, in
//                                                   register r, tile row (r/4)*8 + (l/32)*4 + r%4
//   cols  acc[d][i] += sum_r tile[r][d] w[r][i]     the score registers are the B operand as they
//                                                   are; the tile is read transposed
// bf16 tensors multiply on v_mfma_f32_32x32x16_bf16, fp32 ones on v_mfma_f32_32x32x2_f32 (exact products)
// or, where that pays (attn_train_split), as three bf16 parts each on the former: a = hi + mid + lo holds
// all 24 bits, and the six products down to 2^-16 of the largest leave out what is below 2^-24 of it, at
// 6 x 32 cycles for 16 dims where the fp32 instruction takes 8 x 64.  Sums and softmax statistics are fp32.
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

// What a kernel computes on: the element of its tiles, that of the tensors it writes, and the parts that a
// value is held in.
struct AtF32 {
  typedef float E, O;
  static constexpr int kParts = 1;
};
struct AtBf16 {
  typedef __bf16 E, O;
  static constexpr int kParts = 1;
};
struct AtSplit {
  typedef __bf16 E;
  typedef float O;
  static constexpr int kParts = 3;
};

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

// LDS rows of HD elements in 16-byte chunks, permuted by row.
template <typename E, int HD>
struct AtTile;
template <int HD>
struct AtTile<__bf16, HD> {
  static constexpr int kChunks = HD / 8;
  // the 16 lanes of a 16-byte read (16 rows, one chunk) and the 32 of a transposing read (4 rows, 64 bytes of
  // each) fall on distinct banks
  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (HD == 32) return (row >> 2) & 3;
    if constexpr (HD == 64) return ((row & 2) << 1) | ((row & 4) >> 1) | ((row >> 3) & 1);
    return ((row & 3) << 2) | ((row & 4) >> 1) | ((row >> 3) & 1);
  }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * HD + 8 * (chunk ^ swizzle(row)); }
};
template <int HD>
struct AtTile<float, HD> {
  static constexpr int kChunks = HD / 4;
  // 16 rows of one chunk on distinct banks; the 32 lanes of a column read share a row
  static __device__ __forceinline__ int swizzle(int row) { return HD == 32 ? (row >> 1) & 7 : row & 15; }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * HD + 4 * (chunk ^ swizzle(row)); }
};

// The two products, for heads padded to HD.  A tile of a kind in parts is its parts' tiles, `part` elements
// apart.
template <typename K, int HD>
struct AtMma {
  typedef __bf16 E;
  typedef AtTile<E, HD> L;
  static constexpr int N = K::kParts;
  struct Own {
    at_bf16x8 v[N][HD / 16];  // own row l % 32, dims 16 kk + 8 (l / 32) ..
  };
  template <bool VEC>
  static __device__ __forceinline__ void own(at_bf16x8 (&v)[HD / 16], const AtRows<E>& m, int lane) {
#pragma unroll
    for (int kk = 0; kk < HD / 16; kk++)
      v[kk] = __builtin_bit_cast(at_bf16x8, at_chunk<E, VEC>(m, lane & 31, 2 * kk + (lane >> 5)));
  }
  // a lane's half of the dot product of two own rows
  static __device__ __forceinline__ float dot(const at_bf16x8 (&a)[HD / 16], const at_bf16x8 (&b)[HD / 16]) {
    float s = 0.f;
#pragma unroll
    for (int kk = 0; kk < HD / 16; kk++)
#pragma unroll
      for (int e = 0; e < 8; e++) s = fmaf((float)a[kk][e], (float)b[kk][e], s);
    return s;
  }
  // acc += the products of parts a_i b_j, i + j < N, the small ones first
  static __device__ __forceinline__ void mul(at_f32x16& acc, const at_bf16x8 (&a)[N], const at_bf16x8 (&b)[N]) {
#pragma unroll
    for (int sum = N - 1; sum >= 0; sum--)
#pragma unroll
      for (int i = 0; i <= sum; i++) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[sum - i], acc, 0, 0, 0);
  }
  static __device__ __forceinline__ void rows(at_f32x16& acc, const E* tile, int part, int row0, const Own& o, int lane) {
#pragma unroll
    for (int kk = 0; kk < HD / 16; kk++) {
      at_bf16x8 a[N], b[N];
#pragma unroll
      for (int p = 0; p < N; p++) {
        a[p] = *reinterpret_cast<const at_bf16x8*>(tile + p * part + L::at(row0 + (lane & 31), 2 * kk + (lane >> 5)));
        b[p] = o.v[p][kk];
      }
      mul(acc, a, b);
    }
  }
  // 32 rows of a tile as the operand of `cols`: a transposing read takes 4 rows x 16 dims per 16 lanes; lane
  // i points at 4 dims of row i / 4 and gets dim i of the 4 rows
  static __device__ __forceinline__ at_bf16x8 column(const E* tile, int row0, int kk, int dt, int lane) {
    const int row = row0 + 16 * kk + 4 * (lane >> 5) + ((lane >> 2) & 3);
    const int dim = dt * 32 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    union {
      at_s16x4 h[2];
      at_bf16x8 v;
    } f;
#pragma unroll
    for (int j = 0; j < 2; j++)
      f.h[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) at_s16x4*)(tile + L::at(row + 8 * j, dim >> 3) + (dim & 7)));
    return f.v;
  }
  static constexpr bool kAhead = N == 1 && HD <= 64;  // registers for it before the exponentials
  struct Cols {
    const E* tile;
    int part, row0;
    at_bf16x8 f[kAhead ? 2 : 1][HD / 32];
  };
  static __device__ __forceinline__ Cols load_cols(const E* tile, int part, int row0, int lane) {
    Cols c;
    c.tile = tile, c.part = part, c.row0 = row0;
    if constexpr (kAhead)
#pragma unroll
      for (int kk = 0; kk < 2; kk++)
#pragma unroll
        for (int dt = 0; dt < HD / 32; dt++) c.f[kk][dt] = column(tile, row0, kk, dt, lane);
    return c;
  }
  // w enters a product as the tensors do: rounded to bf16, or in three parts
  static __device__ __forceinline__ void cols(at_f32x16 (&acc)[HD / 32], const Cols& c, const at_f32x16& w, int lane) {
#pragma unroll
    for (int kk = 0; kk < 2; kk++) {
      at_bf16x8 b[N];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        float x = w[8 * kk + e];
#pragma unroll
        for (int p = 0; p < N; p++) {
          b[p][e] = (__bf16)x;
          if (p + 1 < N) x -= (float)b[p][e];
        }
      }
#pragma unroll
      for (int dt = 0; dt < HD / 32; dt++) {
        at_bf16x8 a[N];
#pragma unroll
        for (int p = 0; p < N; p++) a[p] = kAhead ? c.f[kAhead ? kk : 0][dt] : column(c.tile + p * c.part, c.row0, kk, dt, lane);
        mul(acc[dt], a, b);
      }
    }
  }
};

template <int HD>
struct AtMma<AtF32, HD> {
  typedef float E;
  typedef AtTile<E, HD> L;
  struct Own {
    float v[1][HD / 2];  // own row l % 32, dims (l / 32) HD / 2 ..: a product step pairs dims d and d + HD / 2
  };
  template <bool VEC>
  static __device__ __forceinline__ void own(float (&v)[HD / 2], const AtRows<E>& m, int lane) {
#pragma unroll
    for (int c = 0; c < HD / 8; c++) {
      const at_u32x4 x = at_chunk<E, VEC>(m, lane & 31, (lane >> 5) * (HD / 8) + c);
#pragma unroll
      for (int e = 0; e < 4; e++) v[4 * c + e] = __uint_as_float(x[e]);
    }
  }
  static __device__ __forceinline__ float dot(const float (&a)[HD / 2], const float (&b)[HD / 2]) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 2; i++) s = fmaf(a[i], b[i], s);
    return s;
  }
  static __device__ __forceinline__ void rows(at_f32x16& acc, const E* tile, int, int row0, const Own& o, int lane) {
#pragma unroll
    for (int c = 0; c < HD / 8; c++) {
      const float4 a = *reinterpret_cast<const float4*>(tile + L::at(row0 + (lane & 31), (lane >> 5) * (HD / 8) + c));
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, o.v[0][4 * c], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, o.v[0][4 * c + 1], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, o.v[0][4 * c + 2], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, o.v[0][4 * c + 3], acc, 0, 0, 0);
    }
  }
  static constexpr bool kAhead = false;  // (an MFMA takes 64 cycles here and one LDS read)
  struct Cols {
    const E* tile;
  };
  static __device__ __forceinline__ Cols load_cols(const E* tile, int, int row0, int) { return {tile + row0 * HD}; }
  // the tile's rows start at a multiple of 32: of a row's swizzle, bits 2 (HD 32) or 3 (`high`) and up are
  // constants
  static __device__ __forceinline__ void cols(at_f32x16 (&acc)[HD / 32], const Cols& f, const at_f32x16& w, int lane) {
    const int half = lane >> 5, c = (lane & 31) >> 2;
    const E* t = f.tile + 4 * half * HD + (lane & 3);
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int row = (r >> 2) * 8 + (r & 3), high = (r >> 2) & 1;
      const int low = HD == 32 ? (c ^ (2 * half + ((r & 3) >> 1))) ^ (4 * high) : c ^ (4 * half + (r & 3));
#pragma unroll
      for (int dt = 0; dt < HD / 32; dt++)
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(t[row * HD + 4 * low + (HD == 32 ? 0 : 32 * (dt ^ high))], w[r],
                                                       acc[dt], 0, 0, 0);
    }
  }
};

// fp32: 32 rows of m as the operand of `cols`, from memory to registers; zeros past either end of m.
template <int HD>
struct AtColsF32 {
  float v[16][HD / 32];
  __device__ __forceinline__ void load(const AtRows<float>& m, int lane) {
#pragma unroll
    for (int dt = 0; dt < HD / 32; dt++) {
      const int d = dt * 32 + (lane & 31);
      int at = d < m.hd ? 4 * (lane >> 5) * m.stride + 4 * d : 0x7ffffff0;
      asm volatile("" : "+v"(at));  // (or all the loads' offsets are kept in registers from one part to the next)
#pragma unroll
      for (int r = 0; r < 16; r++)
        v[r][dt] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(m.rsrc, at + at_row0(r) * m.stride, 0, 0));
    }
  }
  __device__ __forceinline__ void cols(at_f32x16 (&acc)[HD / 32], const at_f32x16& w) const {
#pragma unroll
    for (int r = 0; r < 16; r++)
#pragma unroll
      for (int dt = 0; dt < HD / 32; dt++) acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[r][dt], w[r], acc[dt], 0, 0, 0);
  }
};

// A matrix in parts: the rows of each, `part` elements (of the whole matrix) apart.
template <typename K>
struct AtSource {
  const typename K::E* base;
  size_t part;
  int stride, hd;  // elements of a row and of a head
  __device__ __forceinline__ AtRows<typename K::E> rows(int p, size_t row, size_t col, int n) const {
    return at_rows(base + p * part + row * stride + col, n, stride, hd);
  }
};
template <typename K, int HD, bool VEC>
__device__ __forceinline__ void at_own(typename AtMma<K, HD>::Own& o, const AtSource<K>& x, size_t row, size_t col, int rows,
                                       int lane) {
#pragma unroll
  for (int p = 0; p < K::kParts; p++) AtMma<K, HD>::template own<VEC>(o.v[p], x.rows(p, row, col, rows), lane);
}

// SR rows of m into an LDS tile, by the block's 256 threads.
template <int HD, int SR, bool VEC, typename E>
__device__ __forceinline__ void at_stage(E* tile, const AtRows<E>& m, int tid) {
  typedef AtTile<E, HD> L;
#pragma unroll
  for (int i = 0; i < SR * L::kChunks / 256; i++) {
    const int row = (tid + 256 * i) / L::kChunks, c = (tid + 256 * i) % L::kChunks;
    *reinterpret_cast<at_u32x4*>(tile + L::at(row, c)) = at_chunk<E, VEC>(m, row, c);
  }
}

// ROWS rows of m straight into an LDS tile: 1 KB pieces (64 lanes x 16 bytes, contiguous in LDS),
// every WAVES-th of them from `first` by this wave.  A lane asks for the chunk whose place is its own.
// Chunks past either end of m arrive as zeros.
template <typename K, int HD, int ROWS, int WAVES>
__device__ __forceinline__ void at_fetch(typename K::E* tile, const AtRows<typename K::E>& m, int first, int lane) {
  typedef typename K::E E;
  typedef AtTile<E, HD> L;
  constexpr int CE = 16 / sizeof(E), RP = 64 / L::kChunks, N = (ROWS / RP + WAVES - 1) / WAVES;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int row0 = (first + WAVES * i) * RP, row = row0 + lane / L::kChunks;
    const int c = (lane % L::kChunks) ^ L::swizzle(row);
    if (ROWS / RP % WAVES == 0 || first + WAVES * i < ROWS / RP)  // (fewer pieces than waves)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(m.rsrc, (__attribute__((address_space(3))) void*)(tile + row0 * HD), 16,
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
// which `rows` exist and the first `len` count: the others are zeros.  RPP > 0: RPP rows at a time by whole
// 16-byte chunks of a row through the wave's part of LDS, `tile` of RPP * HD elements; the pieces that a lane
// holds (4 dims of 32 different rows) would be partial writes of every line (dk and dv of 8 x 1024 bf16 rows:
// 42 us, 35 without the stores).  RPP 0: by the pieces, VEC, or by elements.
template <typename O, int HD, bool VEC, int RPP>
__device__ __forceinline__ void at_store(O* base, int stride, const at_f32x16 (&acc)[HD / 32], float f, int rows, int len,
                                         int hd, O* tile, int lane) {
  typedef AtTile<O, HD> L;
  typedef O o4 __attribute__((ext_vector_type(4)));
  constexpr int CE = 16 / sizeof(O);
  const int i = lane & 31;
  auto each = [&](auto&& put) {
#pragma unroll
    for (int dt = 0; dt < HD / 32; dt++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int dim = dt * 32 + 8 * g + 4 * (lane >> 5);
        o4 v = {(O)(acc[dt][4 * g] * f), (O)(acc[dt][4 * g + 1] * f), (O)(acc[dt][4 * g + 2] * f),
                (O)(acc[dt][4 * g + 3] * f)};
        if (i >= len) v = o4{(O)0.f, (O)0.f, (O)0.f, (O)0.f};
        put(dim, v);
      }
  };
  if constexpr (RPP > 0) {
    constexpr int RP = 64 / L::kChunks;
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += RPP) {
      if (RPP == 32 || (i >= r0 && i < r0 + RPP))
        each([&](int dim, const o4& v) { *reinterpret_cast<o4*>(tile + L::at(i - r0, dim / CE) + dim % CE) = v; });
#pragma unroll
      for (int p = 0; p < RPP / RP; p++) {
        const int row = p * RP + lane / L::kChunks, c = lane % L::kChunks;
        const at_u32x4 v = *reinterpret_cast<const at_u32x4*>(tile + L::at(row, c));
        if (r0 + row < rows && c * CE < hd) *reinterpret_cast<at_u32x4*>(base + (size_t)(r0 + row) * stride + c * CE) = v;
      }
    }
  } else {
    each([&](int dim, const o4& v) {
      O* to = base + (size_t)i * stride + dim;
      if constexpr (VEC) {
        if (i < rows && dim < hd) *reinterpret_cast<o4*>(to) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (i < rows && dim + e < hd) to[e] = v[e];
      }
    });
  }
}

// How a block goes through the axis it walks.
// KS == 1: its four waves own 32 rows each of the other axis and share tiles of kRows rows, which are
// requested one ahead into the other of two buffers (at_walk).
// KS == 4: they own the same 32 rows; each takes every fourth 32-row part through tiles of its own,
// without a barrier, and the sums are joined at the end.  A part's two tiles have one place each: the
// next part's is requested as soon as a tile has been read for the last time, while the products with
// the other one run, so that two blocks fit a CU.
// VEC: rows of 16-byte chunks.
template <typename K, int HD, int KS, bool VEC>
struct AtPlan {
  typedef typename K::E E;
  typedef typename K::O O;
  static constexpr int kOwn = 128 / KS;  // rows of a block
  static constexpr int kRows = KS == 4 || K::kParts > 1 || sizeof(E) * HD > 256 ? 32 : 64;
  static constexpr int kParts = kRows / 32;             // 32-row parts of a tile
  static constexpr int kSub = kRows * HD;               // elements of one part of the values
  static constexpr int kTile = kSub * K::kParts;        // elements of one operand's tile
  static constexpr int kLoads = kTile * (int)sizeof(E) / 1024 / (KS == 4 ? 1 : 4);  // a wave's requests for a tile
  static constexpr int kBufs = VEC && KS == 1 ? 2 : 1;
  static constexpr int kBytes = 2 * kTile * KS * (int)sizeof(E);  // a buffer: both operands, all waves
  // at_store's rows at a time
  static constexpr int kOut = !VEC || KS != 1 ? 0 : 128 * HD * (int)sizeof(O) <= kBytes ? 32
                              : 64 * HD * (int)sizeof(O) <= kBytes ? 16 : 0;
};

// A tile of rows `row` .. of x: by all four waves of the block (KS == 1), or by this wave alone.
template <typename K, int HD, int KS, bool VEC>
__device__ __forceinline__ void at_load(typename K::E* tile, const AtSource<K>& x, size_t row, size_t col, int rows, int w,
                                        int lane) {
  typedef AtPlan<K, HD, KS, VEC> P;
  static_assert(VEC || KS == 1, "element loads are shared by the block");
#pragma unroll
  for (int p = 0; p < K::kParts; p++) {
    const AtRows<typename K::E> m = x.rows(p, row, col, min(rows, P::kRows));
    if constexpr (VEC)
      at_fetch<K, HD, P::kRows, KS == 4 ? 1 : 4>(tile + p * P::kSub, m, KS == 4 ? 0 : w, lane);
    else
      at_stage<HD, P::kRows, false>(tile + p * P::kSub, m, 64 * w + lane);
  }
}

// KS == 1: the steps 0 .. n - 1 of a walk: step kt computes on a buffer whose tiles have landed while those of
// kt + 1 are on their way to the other.  The two buffers are LDS variables of their own and appear by
// name in code of their own, so that the compiler does not make the reads of one wait for the other.  STARTED:
// the caller has requested step 0 (kBufs 2).
template <typename P, bool STARTED = false, typename F, typename C>
__device__ __forceinline__ void at_walk(int n, char* even, char* odd, const F& fetch, const C& compute) {
  if constexpr (P::kBufs == 2) {
    if (!STARTED) fetch(0, even);
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

// Products of a part that crosses the diagonal give masked rows the weight 0, and 0 times an infinity or a NaN
// is a NaN, which belongs to no row that does not see them.  So where a wave's results are not finite, it looks
// at the 32 rows x of its diagonal part: a result that only rows hidden from it can have spoilt is computed
// again from the tensors, adding up only what its row sees.  Lane l has own row l % 32 and dims l / 32 HD / 2 ..
// of it here.  (After the stores, so that nothing of it is in the loops.)
template <int N>
__device__ __forceinline__ bool at_spoilt(const at_f32x16 (&acc)[N]) {
  float s = 0.f;
#pragma unroll
  for (int dt = 0; dt < N; dt++)
#pragma unroll
    for (int r = 0; r < 16; r++) s = fmaf(acc[dt][r], 0.f, s);
  return __builtin_amdgcn_ballot_w64(s != s) != 0;
}
// The same of any wave of a block whose waves have stored parts of the same rows; then those stores have arrived.
__device__ __forceinline__ bool at_block_spoilt(bool spoilt) {
  if (!__syncthreads_or(spoilt)) return false;
  __builtin_amdgcn_s_waitcnt(0x0f70);
  __syncthreads();
  return true;
}
// Whether some dim of the lane's is not finite in a hidden row of x (n rows, stride apart) and finite in all
// that its own row i sees: rows 0 .. i, or (UP) i .. n - 1.
template <typename O, bool UP>
__device__ __forceinline__ bool at_hidden(const O* x, size_t stride, int n, int i, int d0, int dims, int hd) {
  bool need = false;
#pragma unroll 1
  for (int d = d0; d < d0 + dims && d < hd; d++) {
    bool hidden = false, seen = false;
#pragma unroll 1
    for (int r = 0; r < n; r++) {
      const float v = (float)x[r * stride + d];
      const bool bad = !(fabsf(v) < INFINITY), sees = UP ? r >= i : r <= i;
      hidden = hidden || (bad && !sees);
      seen = seen || (bad && sees);
    }
    need = need || (hidden && !seen);
  }
  return __builtin_amdgcn_ballot_w64(need) != 0;
}
template <typename O>
__device__ __forceinline__ float at_dot(const O* x, const O* y, int hd) {
  float s = 0.f;
#pragma unroll 8
  for (int d = 0; d < hd; d++) s = fmaf((float)x[d], (float)y[d], s);
  return s;
}
// acc += w * row[d] over the lane's dims
template <typename O, int N>
__device__ __forceinline__ void at_add_row(float (&acc)[N], float w, const O* row, int d0, int hd) {
#pragma unroll
  for (int d = 0; d < N; d++)
    if (d0 + d < hd) acc[d] = fmaf(w, (float)row[d0 + d], acc[d]);
}
template <typename O, int N>
__device__ __forceinline__ void at_put_row(O* row, const float (&acc)[N], float f, int d0, int hd) {
#pragma unroll
  for (int d = 0; d < N; d++)
    if (d0 + d < hd) row[d0 + d] = (O)(acc[d] * f);
}

// Block -> (block of the axis, group = sequence * heads + head) of a causal launch over nblk * G
// blocks; block 0 of the axis is the one with the most work, and is started first.  Workgroups reach
// the 8 XCDs round-robin.  Sequences of one length: when 8 divides G, an XCD takes whole neighbouring
// groups, so that what their blocks share is fetched into its L2 only.  Every other 32 of its blocks (256 of the
// launch's), one for each CU, come in reverse, so that a CU's blocks add up to the same (dq of 8 x 1024 rows, three
// blocks to a CU: 32.1 -> 30.5 us); `before`: blocks that the launch has before these.  Sequences of their own lengths:
// a group's blocks go to all XCDs in turn, which evens out what long ones cost (4 x up to 1333 rows, 16
// heads of 128, dq: 60 us with groups kept together, an XCD idle for half of it).
struct AtBlock {
  int blk, g;
};
__device__ __forceinline__ AtBlock at_block(int L, int blocks, int before, int G, int ragged) {
  if (ragged) {
    const int blk = L / G, i = L % G;
    return {blk, G % 2 == 0 ? (i + blk) % G : i};
  }
  const bool grouped = G % 8 == 0;
  // place among the blocks of the XCD, or of the launch; 1 << lg of them are one to a CU
  const int i = grouped ? L >> 3 : L, n = grouped ? blocks >> 3 : blocks, off = grouped ? before >> 3 : before;
  const int lg = grouped ? 5 : 8, turn = (i + off) >> lg;
  const int first = max(0, (turn << lg) - off), last = min(n, ((turn + 1) << lg) - off) - 1;
  const int s = turn & 1 ? first + last - i : i, per = grouped ? G / 8 : G;
  return {s / per, grouped ? (L & 7) * per + s % per : s % per};
}

// q's columns of a matrix that a kernel reads (its k and v follow), and do's.
template <typename K>
__device__ __forceinline__ AtSource<K> at_qkv(const AttnTrain& a) {
  return {static_cast<const typename K::E*>(a.in), a.in_part, a.in_cols, a.in_hd};
}
template <typename K>
__device__ __forceinline__ AtSource<K> at_do(const AttnTrain& a) {
  return {static_cast<const typename K::E*>(a.in_do), a.do_part, a.do_cols, a.in_hd};
}

__device__ __forceinline__ int at_len(const AttnTrain& a, int b) {
  if (!a.ragged) return a.T;
  return __builtin_amdgcn_readfirstlane(a.lens_dev ? a.lens_dev[b] : a.lens[b]);
}

}  // namespace fh
