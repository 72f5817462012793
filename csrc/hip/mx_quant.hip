// MXFP4 quantisation and dequantisation (format and layout: mx.h).
#include "mx_common.h"

namespace gpumon_hip {
namespace mx {
namespace {

// Eight elements of a row from column k0 on as words, zeros from column k on. Rows start where the
// caller's stride puts them, so the 16 bytes need not be aligned (one unaligned load).
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int k0, int k, unsigned* w) {
  constexpr int N = 8 / Elem<T>::kPerWord;
  if (k0 + 8 <= k) {
    __builtin_memcpy(w, row + k0, N * 4);
  } else {
    T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k0 + j < k ? row[k0 + j] : T{};
    __builtin_memcpy(w, v, N * 4);
  }
}

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

// Blocks down a column; the result's rows are x's columns. Lanes along the columns, wave w on block w
// of each of a group's four quads: a lane's 32 elements are a block, its four blocks' scales a word.
template <typename T>
__global__ void __launch_bounds__(256) quantize_cols_kernel(const T* __restrict__ x, int64_t stride, unsigned rows,
                                                            unsigned k, Div strips, unsigned quads, unsigned groups,
                                                            char* __restrict__ codes, char* __restrict__ scales) {
  const unsigned g = strips.quot(blockIdx.x), lane = threadIdx.x & 63, b = threadIdx.x >> 6;
  const unsigned c = (blockIdx.x - g * strips.d) * 64 + lane;
  if (c >= (k + 15) / 16 * 16) return;
  unsigned word = 0;
#pragma unroll 1
  for (unsigned j = 0; j < 4 && g * 4 + j < quads; ++j) {
    const unsigned r0 = (g * 4 + j) * 128 + b * 32;
    T v[32];
#pragma unroll
    for (unsigned i = 0; i < 32; ++i)
      v[i] = r0 + i < rows && c < k ? x[static_cast<int64_t>(r0 + i) * stride + c] : T{};
    unsigned w[32 / Elem<T>::kPerWord];
    __builtin_memcpy(w, v, sizeof(w));
    unsigned m = 0;
#pragma unroll
    for (unsigned u : w) m = Elem<T>::amax(m, u);
    const unsigned byte = scale_byte(Elem<T>::amax_f32(m));
    const float s = scale_of(byte);
    u32x4 o;
#pragma unroll
    for (int p = 0; p < 4; ++p) o[p] = byte == 255 ? 0u : codes8<T>(w + p * 8 / Elem<T>::kPerWord, s);
    *reinterpret_cast<u32x4*>(codes + (static_cast<size_t>(c >> 4) * quads + g * 4 + j) * 1024 + b * 256 + (c & 15) * 16) = o;
    word |= byte << (8 * j);
  }
  *reinterpret_cast<unsigned*>(scales + (static_cast<size_t>(c >> 4) * groups + g) * 256 + b * 64 + (c & 15) * 4) = word;
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const char* __restrict__ codes, const char* __restrict__ scales,
                                                         unsigned rows, int k, Div groups, unsigned quads,
                                                         T* __restrict__ out, int64_t stride) {
  __shared__ Piece piece;
  const unsigned rb = groups.quot(blockIdx.x), g = blockIdx.x - rb * groups.d;
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quad = lane >> 4, block = (lane >> 2) & 3;
  if (g * 4 + wave < quads)
    *reinterpret_cast<u32x4*>(&piece.codes[Piece::at(wave, lane >> 4, lane & 15, 0)]) =
        *reinterpret_cast<const u32x4*>(codes + (static_cast<size_t>(rb) * quads + g * 4 + wave) * 1024 + lane * 16);
  if (wave == 0)
    reinterpret_cast<unsigned*>(piece.scales)[lane] =
        *reinterpret_cast<const unsigned*>(scales + (static_cast<size_t>(rb) * groups.d + g) * 256 + lane * 4);
  __syncthreads();
  const int k0 = static_cast<int>(g * 512 + lane * 8);
#pragma unroll
  for (unsigned i = 0; i < 4; ++i) {
    const unsigned r = wave * 4 + i, row = rb * 16 + r;
    if (row >= rows || k0 >= k) return;
    const unsigned c = piece.codes[Piece::at(quad, block, r, lane & 3)];
    const float s = scale_of(piece.scales[(block * 16 + r) * 4 + quad]);
    const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
    const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
    T v[8] = {Elem<T>::from_f32(p0.x), Elem<T>::from_f32(p0.y), Elem<T>::from_f32(p1.x), Elem<T>::from_f32(p1.y),
              Elem<T>::from_f32(p2.x), Elem<T>::from_f32(p2.y), Elem<T>::from_f32(p3.x), Elem<T>::from_f32(p3.y)};
    T* o = out + static_cast<int64_t>(row) * stride + k0;
    if (k0 + 8 <= k) {
      __builtin_memcpy(o, v, sizeof(v));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k0 + j < k) o[j] = v[j];
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
      const unsigned groups = static_cast<unsigned>(mx_groups(rows)), strips = blocks_for(k, 64);
      hipLaunchKernelGGL(quantize_cols_kernel<T>, dim3(groups * strips), dim3(256), 0, s, px, stride,
                         static_cast<unsigned>(rows), static_cast<unsigned>(k), Div(strips),
                         static_cast<unsigned>(mx_quads(rows)), groups, pc, ps);
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
  launch_mx_quantize(dev, x, dtype, rows, k, stride, true, col_codes, col_scales, stream);
  launch_mx_quantize(dev, x, dtype, rows, k, stride, false, row_codes, row_scales, stream);
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
