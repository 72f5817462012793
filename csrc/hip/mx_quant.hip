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
};

// Blocks along a row. A wave takes four rows one after the other (their loads in flight together), 512
// elements of each: 16 lanes a quad, eight elements a lane, so four lanes share a block.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, int64_t stride, unsigned rows,
                                                            int k, Div groups, unsigned quads, char* __restrict__ codes,
                                                            char* __restrict__ scales) {
  __shared__ Piece piece;
  const unsigned rb = groups.quot(blockIdx.x), g = blockIdx.x - rb * groups.d;
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quad = lane >> 4, block = (lane >> 2) & 3;
  unsigned w[4][8 / Elem<T>::kPerWord];
#pragma unroll
  for (unsigned i = 0; i < 4; ++i) {
    const unsigned row = rb * 16 + wave * 4 + i;
    if (row < rows) load8(x + static_cast<int64_t>(row) * stride, static_cast<int>(g * 512 + lane * 8), k, w[i]);
    else
      for (unsigned& v : w[i]) v = 0;
  }
#pragma unroll
  for (unsigned i = 0; i < 4; ++i) {
    unsigned m = 0;
#pragma unroll
    for (unsigned v : w[i]) m = Elem<T>::amax(m, v);
    m = Elem<T>::amax_f32(m);
    m = max(m, dpp<kXor1>(m));
    m = max(m, dpp<kXor2>(m));
    const unsigned byte = scale_byte(m);
    piece.codes[Piece::at(quad, block, wave * 4 + i, lane & 3)] = byte == 255 ? 0u : codes8<T>(w[i], scale_of(byte));
    if ((lane & 3) == 0) piece.scales[(block * 16 + wave * 4 + i) * 4 + quad] = static_cast<unsigned char>(byte);
  }
  __syncthreads();
  if (g * 4 + wave < quads)
    *reinterpret_cast<u32x4*>(codes + (static_cast<size_t>(rb) * quads + g * 4 + wave) * 1024 + lane * 16) =
        *reinterpret_cast<const u32x4*>(&piece.codes[Piece::at(wave, lane >> 4, lane & 15, 0)]);
  if (wave == 0)
    *reinterpret_cast<unsigned*>(scales + (static_cast<size_t>(rb) * groups.d + g) * 256 + lane * 4) =
        reinterpret_cast<const unsigned*>(piece.scales)[lane];
}

// Blocks down a column (the result's rows are x's columns), and with ROWS along the rows too, from one
// reading. A workgroup takes 128 x 128 elements: as they arrive, 16 lanes on a row's quad, they are
// quantised along the row and left in LDS; then wave b takes block b of every column, a lane two
// columns of a 16-bit type (a word of each of 32 rows) or one and then another of f32.
template <typename T, bool ROWS>
__global__ void __launch_bounds__(256) quantize_tile_kernel(const T* __restrict__ x, int64_t stride, unsigned rows,
                                                            int k, Div tiles_k, char* __restrict__ row_codes,
                                                            char* __restrict__ row_scales, char* __restrict__ col_codes,
                                                            char* __restrict__ col_scales) {
  constexpr int kWords = 8 / Elem<T>::kPerWord;  // of eight elements
  constexpr int kRow = 16 * kWords;              // words of a row of the tile
  __shared__ __attribute__((aligned(16))) unsigned tile[128 * kRow];
  const unsigned tr = tiles_k.quot(blockIdx.x), tc = blockIdx.x - tr * tiles_k.d;
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, block = l >> 2;
  const unsigned row_groups = (tiles_k.d + 3) / 4, quads = (rows + 127) / 128, col_groups = (quads + 3) / 4;
  unsigned w[8][kWords];
#pragma unroll
  for (unsigned i = 0; i < 8; ++i) {
    const unsigned row = tr * 128 + wave * 32 + i * 4 + (lane >> 4);
    if (row < rows) load8(x + static_cast<int64_t>(row) * stride, static_cast<int>(tc * 128 + l * 8), k, w[i]);
    else
      for (unsigned& v : w[i]) v = 0;
  }
#pragma unroll
  for (unsigned i = 0; i < 8; ++i) {
    const unsigned r = wave * 32 + i * 4 + (lane >> 4), row = tr * 128 + r;
#pragma unroll
    for (int p = 0; p < kWords; p += 4)
      *reinterpret_cast<u32x4*>(&tile[r * kRow + l * kWords + p]) = u32x4{w[i][p], w[i][p + 1], w[i][p + 2], w[i][p + 3]};
    if constexpr (ROWS) {
      unsigned m = 0;
#pragma unroll
      for (unsigned v : w[i]) m = Elem<T>::amax(m, v);
      m = Elem<T>::amax_f32(m);
      m = max(m, dpp<kXor1>(m));
      m = max(m, dpp<kXor2>(m));
      const unsigned byte = scale_byte(m);
      const unsigned c = byte == 255 ? 0u : codes8<T>(w[i], scale_of(byte));
      if ((row >> 4) < (rows + 15) >> 4) {
        *reinterpret_cast<unsigned*>(row_codes + (static_cast<size_t>(row >> 4) * tiles_k.d + tc) * 1024 + block * 256 +
                                     (row & 15) * 16 + (l & 3) * 4) = c;
        if ((l & 3) == 0) {
          char* s = row_scales + (static_cast<size_t>(row >> 4) * row_groups + (tc >> 2)) * 256 + block * 64 + (row & 15) * 4;
          s[tc & 3] = static_cast<char>(byte);
          if (tc + 1 == tiles_k.d)
            for (unsigned j = (tc & 3) + 1; j < 4; ++j) s[j] = 0;
        }
      }
    }
  }
  __syncthreads();
  auto store = [&](unsigned col, const unsigned* v) {  // 32 elements of a column
    if (static_cast<int>(col) >= (k + 15) / 16 * 16) return;
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 32 / Elem<T>::kPerWord; ++i) m = Elem<T>::amax(m, v[i]);
    const unsigned byte = scale_byte(Elem<T>::amax_f32(m));
    const float s = scale_of(byte);
    u32x4 o;
#pragma unroll
    for (int p = 0; p < 4; ++p) o[p] = byte == 255 ? 0u : codes8<T>(v + p * kWords, s);
    *reinterpret_cast<u32x4*>(col_codes + (static_cast<size_t>(col >> 4) * quads + tr) * 1024 + wave * 256 + (col & 15) * 16) = o;
    char* sp = col_scales + (static_cast<size_t>(col >> 4) * col_groups + (tr >> 2)) * 256 + wave * 64 + (col & 15) * 4;
    sp[tr & 3] = static_cast<char>(byte);
    if (tr + 1 == quads)
      for (unsigned j = (tr & 3) + 1; j < 4; ++j) sp[j] = 0;
  };
  if constexpr (Elem<T>::kPerWord == 2) {
    unsigned lo[16], hi[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const unsigned a = tile[(wave * 32 + 2 * i) * kRow + lane], b = tile[(wave * 32 + 2 * i + 1) * kRow + lane];
      lo[i] = (a & 0xffffu) | (b << 16);
      hi[i] = (a >> 16) | (b & 0xffff0000u);
    }
    store(tc * 128 + lane * 2, lo);
    store(tc * 128 + lane * 2 + 1, hi);
  } else {
#pragma unroll 1
    for (unsigned h = 0; h < 2; ++h) {
      unsigned v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = tile[(wave * 32 + i) * kRow + h * 64 + lane];
      store(tc * 128 + h * 64 + lane, v);
    }
  }
}

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
  // 16 bytes a lane and store, next to each other: eight elements of a 16-bit type, four of f32
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
      store16(o, v);
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

template <typename T, bool ROWS>
void launch_tiles(const T* x, int64_t rows, int64_t k, int64_t stride, char* row_codes, char* row_scales,
                  char* col_codes, char* col_scales, hipStream_t s) {
  const unsigned tiles_k = static_cast<unsigned>(mx_quads(k));
  hipLaunchKernelGGL((quantize_tile_kernel<T, ROWS>), dim3(tiles_k * static_cast<unsigned>(mx_quads(rows))), dim3(256), 0, s,
                     x, stride, static_cast<unsigned>(rows), static_cast<int>(k), Div(tiles_k), row_codes, row_scales,
                     col_codes, col_scales);
}

}  // namespace
}  // namespace mx

using namespace mx;

void launch_mx_quantize(int dev, const void* x, const std::string& dtype, int64_t rows, int64_t k, int64_t stride,
                        bool by_column, void* codes, void* scales, void* stream) {
  const Type t = type_of(dtype, "mx_quantize: dtype must be bf16|f16|f32");
  check_matrix(x, rows, k, stride, codes, scales, t);
  if (by_column) {
    require(rows >= 1, "mx_quantize: by column, rows must be >= 1");
    check_matrix(x, k, rows, rows, codes, scales, t);
  }
  if (rows == 0) return;
  OnDevice on(dev);
  auto s = static_cast<hipStream_t>(stream);
  auto pc = static_cast<char*>(codes), ps = static_cast<char*>(scales);
  with_type(t, [&](auto e) {
    using T = decltype(e);
    auto px = static_cast<const T*>(x);
    if (by_column) {
      launch_tiles<T, false>(px, rows, k, stride, nullptr, nullptr, pc, ps, s);
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
  check_matrix(x, rows, k, stride, row_codes, row_scales, t);
  require(rows >= 1, "mx_quantize_both: rows must be >= 1");
  check_matrix(x, k, rows, rows, col_codes, col_scales, t);
  OnDevice on(dev);
  with_type(t, [&](auto e) {
    using T = decltype(e);
    launch_tiles<T, true>(static_cast<const T*>(x), rows, k, stride, static_cast<char*>(row_codes),
                          static_cast<char*>(row_scales), static_cast<char*>(col_codes), static_cast<char*>(col_scales),
                          static_cast<hipStream_t>(stream));
  });
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
