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

// Blocks along a row: 16 lanes take a quad, eight elements each, so four lanes share a block.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, int64_t stride, unsigned rows,
                                                            int k, Div quads, unsigned units,
                                                            unsigned* __restrict__ codes, unsigned* __restrict__ scales) {
  const unsigned unit = blockIdx.x * 16 + (threadIdx.x >> 4), l = threadIdx.x & 15;
  if (unit >= units) return;
  const unsigned row = quads.quot(unit), q = unit - row * quads.d;
  unsigned w[8 / Elem<T>::kPerWord];
  load8(x + static_cast<int64_t>(row) * stride, static_cast<int>(q * 128 + l * 8), k, w);
  unsigned m = 0;
#pragma unroll
  for (unsigned v : w) m = Elem<T>::amax(m, v);
  m = Elem<T>::amax_f32(m);
  m = max(m, dpp<kXor1>(m));
  m = max(m, dpp<kXor2>(m));
  const unsigned byte = scale_byte(m);
  const unsigned c = byte == 255 ? 0u : codes8<T>(w, scale_of(byte));
  codes[static_cast<size_t>(unit) * 16 + l] = c;
  unsigned word = byte << (8 * (l >> 2));
  word |= dpp<kRor4>(word);
  word |= dpp<kRor8>(word);
  if (l == 0) scales[static_cast<size_t>(q) * rows + row] = word;
}

// Blocks down a column: lanes along the columns, one block of 32 rows a lane, the four waves of a
// workgroup on the four blocks of a quad. The result's rows are x's columns.
template <typename T>
__global__ void __launch_bounds__(256) quantize_cols_kernel(const T* __restrict__ x, int64_t stride, unsigned rows,
                                                            unsigned k, Div strips, unsigned* __restrict__ codes,
                                                            unsigned* __restrict__ scales, unsigned quads) {
  __shared__ unsigned char sb[64][4];
  const unsigned q = strips.quot(blockIdx.x), lane = threadIdx.x & 63, b = threadIdx.x >> 6;
  const unsigned c = (blockIdx.x - q * strips.d) * 64 + lane;
  if (c < k) {
    const unsigned r0 = q * 128 + b * 32;
    T v[32];
#pragma unroll
    for (unsigned i = 0; i < 32; ++i)
      v[i] = r0 + i < rows ? x[static_cast<int64_t>(r0 + i) * stride + c] : T{};
    unsigned w[32 / Elem<T>::kPerWord];
    __builtin_memcpy(w, v, sizeof(w));
    unsigned m = 0;
#pragma unroll
    for (unsigned u : w) m = Elem<T>::amax(m, u);
    const unsigned byte = scale_byte(Elem<T>::amax_f32(m));
    const float s = scale_of(byte);
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = byte == 255 ? 0u : codes8<T>(w + j * 8 / Elem<T>::kPerWord, s);
    *reinterpret_cast<u32x4*>(codes + (static_cast<size_t>(c) * quads + q) * 16 + b * 4) = o;
    sb[lane][b] = static_cast<unsigned char>(byte);
  }
  __syncthreads();
  if (b == 0 && c < k)
    scales[static_cast<size_t>(q) * k + c] = *reinterpret_cast<const unsigned*>(sb[lane]);
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const unsigned* __restrict__ codes,
                                                         const unsigned* __restrict__ scales, unsigned rows, int k,
                                                         Div quads, unsigned units, T* __restrict__ out, int64_t stride) {
  const unsigned unit = blockIdx.x * 16 + (threadIdx.x >> 4), l = threadIdx.x & 15;
  if (unit >= units) return;
  const unsigned row = quads.quot(unit), q = unit - row * quads.d;
  const unsigned c = codes[static_cast<size_t>(unit) * 16 + l];
  const float s = scale_of((scales[static_cast<size_t>(q) * rows + row] >> (8 * (l >> 2))) & 255);
  const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
  const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
  T v[8] = {Elem<T>::from_f32(p0.x), Elem<T>::from_f32(p0.y), Elem<T>::from_f32(p1.x), Elem<T>::from_f32(p1.y),
            Elem<T>::from_f32(p2.x), Elem<T>::from_f32(p2.y), Elem<T>::from_f32(p3.x), Elem<T>::from_f32(p3.y)};
  const int k0 = static_cast<int>(q * 128 + l * 8);
  T* o = out + static_cast<int64_t>(row) * stride + k0;
  if (k0 + 8 <= k) {
    __builtin_memcpy(o, v, sizeof(v));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k0 + j < k) o[j] = v[j];
  }
}

// What the kernels' 31-bit indexes and grids hold.
void check_matrix(const void* data, int64_t rows, int64_t k, int64_t stride, const void* codes, const void* scales,
                  Type t) {
  require(rows >= 0 && k >= 1, "mx: rows must be >= 0 and k >= 1");
  require(rows < (1ll << 31) && k <= (1ll << 31) - 256 && rows * mx_quads(k) < (1ll << 31),
          "mx: rows, k and rows * ceil(k / 128) must be below 2^31");
  require(stride >= k || rows <= 1, "mx: stride must be at least k");
  if (rows == 0) return;
  require(data && codes && scales, "mx: null pointer");
  require(aligned(data, size_of(t)) && aligned(codes, 16) && aligned(scales, 4),
          "mx: data aligned to its type, codes to 16 and scales to 4 bytes");
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
  auto pc = static_cast<unsigned*>(codes), ps = static_cast<unsigned*>(scales);
  with_type(t, [&](auto e) {
    using T = decltype(e);
    auto px = static_cast<const T*>(x);
    if (by_column) {
      const unsigned quads = static_cast<unsigned>(mx_quads(rows)), strips = blocks_for(k, 64);
      hipLaunchKernelGGL(quantize_cols_kernel<T>, dim3(quads * strips), dim3(256), 0, s, px, stride,
                         static_cast<unsigned>(rows), static_cast<unsigned>(k), Div(strips), pc, ps, quads);
    } else {
      const unsigned units = static_cast<unsigned>(rows * mx_quads(k));
      hipLaunchKernelGGL(quantize_rows_kernel<T>, dim3(blocks_for(units, 16)), dim3(256), 0, s, px, stride,
                         static_cast<unsigned>(rows), static_cast<int>(k), Div(static_cast<unsigned>(mx_quads(k))), units,
                         pc, ps);
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
  const unsigned units = static_cast<unsigned>(rows * mx_quads(k));
  with_type(t, [&](auto e) {
    using T = decltype(e);
    hipLaunchKernelGGL(dequantize_kernel<T>, dim3(blocks_for(units, 16)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const unsigned*>(codes), static_cast<const unsigned*>(scales),
                       static_cast<unsigned>(rows), static_cast<int>(k), Div(static_cast<unsigned>(mx_quads(k))), units,
                       static_cast<T*>(out), stride);
  });
  check(hipGetLastError(), "mx_dequantize");
}

}  // namespace gpumon_hip
