// MXFP4 quantisation and dequantisation (format and layout: mx.h).
#include "mx_common.h"

namespace gpumon_hip {
namespace mx {
namespace {

// A workgroup's piece of a quantised matrix, 16 rows x 4 quads, in LDS: codes with the rows of each
// block rotated (writers of different blocks and quads would all meet in four banks), scales as they
// are in memory.
struct Piece {
  __attribute__((aligned(16))) unsigned codes[1024];
  __attribute__((aligned(16))) unsigned char scales[256];
  // word w of the block's 16 bytes
  __device__ static unsigned at(unsigned quad, unsigned block, unsigned row, unsigned w) {
    return quad * 256 + block * 64 + ((row + block + 4 * quad) & 15) * 4 + w;
  }
  // A wave's 512 elements of a row, eight a lane: 16 lanes a quad, so four lanes share a block.
  template <typename T>
  __device__ __forceinline__ void put(const unsigned* w, unsigned row, unsigned lane) {
    const unsigned quad = lane >> 4, block = (lane >> 2) & 3;
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8 / Elem<T>::kPerWord; ++i) m = Elem<T>::amax(m, w[i]);
    m = Elem<T>::amax_f32(m);
    m = max(m, dpp<kXor1>(m));
    m = max(m, dpp<kXor2>(m));
    const unsigned byte = scale_byte(m);
    codes[at(quad, block, row, lane & 3)] = byte == 255 ? 0u : codes8<T>(w, scale_of(byte));
    if ((lane & 3) == 0) scales[(block * 16 + row) * 4 + quad] = static_cast<unsigned char>(byte);
  }
  // By four waves, to row block rb and group g.
  __device__ __forceinline__ void store(char* out, char* out_scales, unsigned rb, unsigned g, unsigned quads, unsigned groups) const {
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6 & 3;
    if (g * 4 + wave < quads)
      *reinterpret_cast<u32x4*>(out + (static_cast<size_t>(rb) * quads + g * 4 + wave) * 1024 + lane * 16) =
          *reinterpret_cast<const u32x4*>(&codes[at(wave, lane >> 4, lane & 15, 0)]);
    if (wave == 0)
      *reinterpret_cast<unsigned*>(out_scales + (static_cast<size_t>(rb) * groups + g) * 256 + lane * 4) =
          reinterpret_cast<const unsigned*>(scales)[lane];
  }
};

// Blocks along a row: amax, the scale's exponent and the codes as in mx.h. A wave takes 512 elements of four
// rows, their loads in flight together; a workgroup ends up with whole chunks and scale words and writes
// them 16 bytes a lane. Bound by memory: 8192 x 8192 bf16 (134 MB read, 36 written) 28.7 us, 5.9 TB/s,
// where a plain copy of 1 GiB reaches 6.54; one token of 8192 2.8 us, a launch's least.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, int64_t stride, unsigned rows,
                                                            int k, Div groups, unsigned quads, char* __restrict__ codes,
                                                            char* __restrict__ scales) {
  __shared__ Piece piece;
  const unsigned rb = groups.quot(blockIdx.x), g = blockIdx.x - rb * groups.d;
  const unsigned lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  unsigned w[4][8 / Elem<T>::kPerWord];
  with_reach<T>(static_cast<int>(g * 512 + 512), k, [&](auto how) {
#pragma unroll
    for (unsigned i = 0; i < 4; ++i)
      load8<decltype(how)::value>(x + static_cast<int64_t>(min(rb * 16 + wave * 4 + i, rows - 1)) * stride,
                                  static_cast<int>(g * 512 + lane * 8), k, w[i]);
  });
#pragma unroll
  for (unsigned i = 0; i < 4; ++i) {
    if (rb * 16 + wave * 4 + i >= rows)
      for (unsigned& v : w[i]) v = 0;
    piece.template put<T>(w[i], wave * 4 + i, lane);
  }
  __syncthreads();
  piece.store(codes, scales, rb, g, quads, groups.d);
}

// Blocks down a column (the result's rows are x's columns), and with ROWS along the rows too, from one
// reading. A workgroup takes 32 rows x 512 columns, whole KiB of a row of a 16-bit type at a time: as they
// arrive they are quantised along the row, as above, and left in LDS; then each thread takes a column.
// Both directions of 8192 x 8192 bf16: 40 us, 5.1 TB/s (57 with a wave's loads one after the other, where
// 128 x 128 elements a workgroup took 53). A scale word's four bytes come from four workgroups, each
// storing its own. Bound by memory, and by the chain of its steps where there are few workgroups: both
// directions of two matrices of 4096 x 8192 in one launch 35 us, 5.9 TB/s; of 613 x 1000 f16 4.7 us.
// One launch takes up to two matrices.
struct Both {
  const void* x;
  int64_t stride;
  unsigned rows;
  int k;
  Div groups;
  unsigned blocks;  // workgroups
  char *row_codes, *row_scales, *col_codes, *col_scales;
};
struct TwoBoth {
  Both of[2];
};
template <typename T, bool ROWS>
__global__ void __launch_bounds__(512) quantize_tile_kernel(TwoBoth both) {
  constexpr int kWords = 8 / Elem<T>::kPerWord;  // of eight elements
  constexpr int kRow = 64 * kWords;              // words of a row of the tile
  __shared__ __attribute__((aligned(16))) unsigned tile[32 * kRow];
  __shared__ Piece piece[ROWS ? 2 : 1];
  const Both& m = both.of[blockIdx.x < both.of[0].blocks ? 0 : 1];
  const T* x = static_cast<const T*>(m.x);
  const int64_t stride = m.stride;
  const unsigned rows = m.rows, bid = blockIdx.x - (blockIdx.x < both.of[0].blocks ? 0 : both.of[0].blocks);
  const int k = m.k;
  const Div groups = m.groups;
  char *row_codes = m.row_codes, *row_scales = m.row_scales, *col_codes = m.col_codes, *col_scales = m.col_scales;
  const unsigned tr = groups.quot(bid), g = bid - tr * groups.d;
  const unsigned lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  unsigned w[4][kWords];
  with_reach<T>(static_cast<int>(g * 512 + 512), k, [&](auto how) {
#pragma unroll
    for (unsigned i = 0; i < 4; ++i)
      load8<decltype(how)::value>(x + static_cast<int64_t>(min(tr * 32 + wave * 4 + i, rows - 1)) * stride,
                                  static_cast<int>(g * 512 + lane * 8), k, w[i]);
  });
#pragma unroll
  for (unsigned i = 0; i < 4; ++i) {
    const unsigned r = wave * 4 + i;
    if (tr * 32 + r >= rows)
      for (unsigned& v : w[i]) v = 0;
#pragma unroll
    for (int p = 0; p < kWords; p += 4)
      *reinterpret_cast<u32x4*>(&tile[r * kRow + lane * kWords + p]) = u32x4{w[i][p], w[i][p + 1], w[i][p + 2], w[i][p + 3]};
    if constexpr (ROWS) piece[r >> 4].template put<T>(w[i], r & 15, lane);
  }
  __syncthreads();
  if constexpr (ROWS) {
    const unsigned h = wave >> 2;
    if (tr * 2 + h < (rows + 15) / 16)
      piece[h].store(row_codes, row_scales, tr * 2 + h, g, (static_cast<unsigned>(k) + 127) / 128, groups.d);
  }
  // a column a thread; of a 16-bit type its half of the words that hold two, even columns first
  constexpr int kColWords = 32 / Elem<T>::kPerWord;
  unsigned v[kColWords];
  unsigned c = threadIdx.x;
  if constexpr (Elem<T>::kPerWord == 2) {
    const unsigned pair = threadIdx.x & 255, odd = threadIdx.x >> 8;
    c = pair * 2 + odd;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const unsigned a = tile[2 * i * kRow + pair], b = tile[(2 * i + 1) * kRow + pair];
      v[i] = __builtin_amdgcn_perm(b, a, odd ? 0x07060302u : 0x05040100u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = tile[i * kRow + threadIdx.x];
  }
  unsigned top = 0;
#pragma unroll
  for (unsigned e : v) top = Elem<T>::amax(top, e);
  const unsigned byte = scale_byte(Elem<T>::amax_f32(top));
  const float s = scale_of(byte);
  u32x4 o;
#pragma unroll
  for (int p = 0; p < 4; ++p) o[p] = byte == 255 ? 0u : codes8<T>(v + p * kWords, s);
  // row tr of tiles is block tr % 4 of quad tr / 4 down the columns
  const unsigned quads = (rows + 127) / 128, q = tr >> 2, b = tr & 3, col_groups = (quads + 3) / 4, col = g * 512 + c;
  if (col < (static_cast<unsigned>(k) + 15) / 16 * 16) {
    *reinterpret_cast<u32x4*>(col_codes + (static_cast<size_t>(col >> 4) * quads + q) * 1024 + b * 256 + (col & 15) * 16) = o;
    char* sp = col_scales + (static_cast<size_t>(col >> 4) * col_groups + (q >> 2)) * 256 + b * 64 + (col & 15) * 4;
    sp[q & 3] = static_cast<char>(byte);
    if (q + 1 == quads)
      for (unsigned j = (q & 3) + 1; j < 4; ++j) sp[j] = 0;
  }
}

// Codes times scale, rounded to T (exact in bf16 and f32). The same pieces the other way round; stores past
// the caches: 8192 x 8192 to bf16 25.4 us, 6.7 TB/s (in a graph of several 27.3, and 35.3 with plain
// stores). Rows that do not start on a cache line leave parts of lines at each piece's ends: 4099 x 2053 to
// f32 8.5 us, 4.5 TB/s (in a graph 9.8).
template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const char* __restrict__ codes, const char* __restrict__ scales,
                                                         unsigned rows, int k, Div groups, unsigned quads,
                                                         T* __restrict__ out, int64_t stride) {
  __shared__ Piece piece;
  const unsigned rb = groups.quot(blockIdx.x), g = blockIdx.x - rb * groups.d;
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (g * 4 + wave < quads)
    *reinterpret_cast<u32x4*>(&piece.codes[Piece::at(wave, lane >> 4, lane & 15, 0)]) =
        *reinterpret_cast<const u32x4*>(codes + (static_cast<size_t>(rb) * quads + g * 4 + wave) * 1024 + lane * 16);
  if (wave == 0)
    reinterpret_cast<unsigned*>(piece.scales)[lane] =
        *reinterpret_cast<const unsigned*>(scales + (static_cast<size_t>(rb) * groups.d + g) * 256 + lane * 4);
  __syncthreads();
  // 16 bytes a lane and store, next to each other: eight elements of a 16-bit type, four of f32. Past the
  // caches, but for f32 rows off the lines (4099 x 2053: 11.2 us past them, 9.9 through; 4099 x 2048 7.7 and
  // 8.9; to bf16 8192 x 8191 38 and 50, 8192 x 8192 27 and 35).
  const bool past = sizeof(T) == 2 || whole_lines(out, stride);
  constexpr unsigned kPer = 16 / sizeof(T), kPasses = 8 / kPer;
#pragma unroll
  for (unsigned i = 0; i < 4 * kPasses; ++i) {
    const unsigned r = wave * 4 + i / kPasses, row = rb * 16 + r, e = i % kPasses * 64 * kPer + lane * kPer;
    const int k0 = static_cast<int>(g * 512 + e);
    if (row >= rows || k0 >= k) continue;
    const unsigned quad = e >> 7, block = (e >> 5) & 3;
    const unsigned c = piece.codes[Piece::at(quad, block, r, (e >> 3) & 3)] >> (kPer == 4 ? (e & 4) * 4 : 0);
    const float s = scale_of(piece.scales[(block * 16 + r) * 4 + quad]);
    T v[kPer];
    f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0);
    v[0] = Elem<T>::from_f32(p.x), v[1] = Elem<T>::from_f32(p.y);
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
    v[2] = Elem<T>::from_f32(p.x), v[3] = Elem<T>::from_f32(p.y);
    if constexpr (kPer == 8) {
      p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2);
      v[4] = Elem<T>::from_f32(p.x), v[5] = Elem<T>::from_f32(p.y);
      p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
      v[6] = Elem<T>::from_f32(p.x), v[7] = Elem<T>::from_f32(p.y);
    }
    T* o = out + static_cast<int64_t>(row) * stride + k0;
    if (k0 + static_cast<int>(kPer) <= k) {
      store16(o, v, past);
    } else {
#pragma unroll
      for (unsigned j = 0; j < kPer; ++j)
        if (k0 + static_cast<int>(j) < k) o[j] = v[j];
    }
  }
}

void check_matrix(const void* data, int64_t rows, int64_t k, int64_t stride, const void* codes, const void* scales,
                  Type t) {
  require(rows >= 0 && k >= 1, "mx: rows must be >= 0 and k >= 1");
  require(mx_fits(rows, k), "mx: rows and k are beyond the limits (mx.h)");
  require(stride >= k || rows <= 1, "mx: stride must be at least k");
  if (rows == 0) return;
  require(data && codes && scales, "mx: null pointer");
  require(aligned(data, size_of(t)) && aligned(codes, 16) && aligned(scales, 16),
          "mx: data aligned to its type, codes and scales to 16 bytes");
}

unsigned blocks_for(int64_t n, int64_t per) { return static_cast<unsigned>((n + per - 1) / per); }

unsigned tiles_of(const Both* of, int count) { return of[0].blocks + (count > 1 ? of[1].blocks : 0); }

template <typename T, bool ROWS>
void launch_tiles(const Both* of, int count, hipStream_t s) {
  const TwoBoth both{{of[0], of[count - 1]}};
  hipLaunchKernelGGL((quantize_tile_kernel<T, ROWS>), dim3(tiles_of(of, count)), dim3(512), 0, s, both);
}
Both both_of(const void* x, int64_t rows, int64_t k, int64_t stride, void* rc, void* rs, void* cc, void* cs) {
  const unsigned groups = static_cast<unsigned>(mx_groups(k));
  return {x, stride, static_cast<unsigned>(rows), static_cast<int>(k), Div(groups), static_cast<unsigned>(mx_quads(rows) * 4) * groups,
          static_cast<char*>(rc), static_cast<char*>(rs), static_cast<char*>(cc), static_cast<char*>(cs)};
}
// A launch has fewer than 2^32 threads.
bool fits_launch(int64_t rows, int64_t k) { return mx_quads(rows) * 4 * mx_groups(k) < (1ll << 23); }
void check_both(const void* x, int64_t rows, int64_t k, int64_t stride, const void* row_codes, const void* row_scales,
                const void* col_codes, const void* col_scales, Type t) {
  check_matrix(x, rows, k, stride, row_codes, row_scales, t);
  require(rows >= 1, "mx: down the columns, rows must be >= 1");
  check_matrix(x, k, rows, rows, col_codes, col_scales, t);
  require(fits_launch(rows, k), "mx: rows and k are beyond the limits (mx.h)");
}

}  // namespace

void check_source(const Source& s, Type t) {
  check_both(s.x, s.rows, s.k, s.stride, s.along, s.along, s.down, s.down, t);
}
void launch_quantize_both(int dev, const Source* sources, int count, Type t, hipStream_t s) {
  Both of[2];
  for (int i = 0; i < count; ++i) {
    const Source& m = sources[i];
    const Quantized along{m.along, m.rows, m.k}, down{m.down, m.k, m.rows};
    of[i] = both_of(m.x, m.rows, m.k, m.stride, along.at, along.scales(), down.at, down.scales());
  }
  OnDevice on(dev);
  with_type(t, [&](auto e) {
    using T = decltype(e);
    if (count == 2 && tiles_of(of, 2) >= 1u << 23) {
      launch_tiles<T, true>(of, 1, s);
      launch_tiles<T, true>(of + 1, 1, s);
    } else {
      launch_tiles<T, true>(of, count, s);
    }
  });
  check(hipGetLastError(), "mx_quantize_both");
}

}  // namespace mx

using namespace mx;

void launch_mx_quantize(int dev, const void* x, const std::string& dtype, int64_t rows, int64_t k, int64_t stride,
                        bool by_column, void* codes, void* scales, void* stream) {
  const Type t = type_of(dtype, "mx_quantize: dtype must be bf16|f16|f32");
  if (by_column) check_both(x, rows, k, stride, codes, scales, codes, scales, t);
  else check_matrix(x, rows, k, stride, codes, scales, t);
  if (rows == 0) return;
  auto s = static_cast<hipStream_t>(stream);
  auto pc = static_cast<char*>(codes), ps = static_cast<char*>(scales);
  OnDevice on(dev);
  with_type(t, [&](auto e) {
    using T = decltype(e);
    auto px = static_cast<const T*>(x);
    if (by_column) {
      const Both of = both_of(x, rows, k, stride, nullptr, nullptr, pc, ps);
      launch_tiles<T, false>(&of, 1, s);
    } else {
      const unsigned groups = static_cast<unsigned>(mx_groups(k));
      hipLaunchKernelGGL(quantize_rows_kernel<T>, dim3(groups * blocks_for(rows, 16)), dim3(256), 0, s, px, stride,
                         static_cast<unsigned>(rows), static_cast<int>(k), Div(groups),
                         static_cast<unsigned>(mx_quads(k)), pc, ps);
    }
  });
  check(hipGetLastError(), "mx_quantize");
}

void launch_mx_quantize_both(int dev, const void* x, const std::string& dtype, int64_t rows, int64_t k, int64_t stride,
                             void* row_codes, void* row_scales, void* col_codes, void* col_scales, void* stream) {
  const Type t = type_of(dtype, "mx_quantize_both: dtype must be bf16|f16|f32");
  check_both(x, rows, k, stride, row_codes, row_scales, col_codes, col_scales, t);
  OnDevice on(dev);
  const Both of = both_of(x, rows, k, stride, row_codes, row_scales, col_codes, col_scales);
  with_type(t, [&](auto e) { launch_tiles<decltype(e), true>(&of, 1, static_cast<hipStream_t>(stream)); });
  check(hipGetLastError(), "mx_quantize_both");
}

void launch_mx_dequantize(int dev, const void* codes, const void* scales, int64_t rows, int64_t k, void* out,
                          const std::string& dtype, int64_t stride, void* stream) {
  const Type t = type_of(dtype, "mx_dequantize: dtype must be bf16|f16|f32");
  check_matrix(out, rows, k, stride, codes, scales, t);
  if (rows == 0) return;
  OnDevice on(dev);
  const unsigned groups = static_cast<unsigned>(mx_groups(k));
  with_type(t, [&](auto e) {
    using T = decltype(e);
    hipLaunchKernelGGL(dequantize_kernel<T>, dim3(groups * blocks_for(rows, 16)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), static_cast<const char*>(codes), static_cast<const char*>(scales),
                       static_cast<unsigned>(rows), static_cast<int>(k), Div(groups), static_cast<unsigned>(mx_quads(k)),
                       static_cast<T*>(out), stride);
  });
  check(hipGetLastError(), "mx_dequantize");
}

}  // namespace gpumon_hip
