// MXFP4 operators: quantisation, product and linear layer (mx_quant.hip, mx_product.hip).
//
// Format. A matrix of `rows` x `k` is held in blocks of 32 consecutive elements of a row: 4 bits an
// element (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) and one scale byte a block (e8m0:
// 2^(byte - 127); 255: the block stands for NaN). With amax the block's largest magnitude,
//     E = clamp(floor(log2 amax) - 2, -127, 125)   (amax = 0: -127),   byte = E + 127,
//     q_i = x_i / 2^E rounded to the grid, halves to the even code, beyond 6 to 6;
// a NaN or an infinity in the block: byte 255. Dividing by 2^E is exact, so every code is determined.
//
// Layout. k is filled up with zeros to whole "quads" of 128 elements, kq = ceil(k / 128):
//     codes  [rows][kq * 64] bytes, the even element in the low nibble;
//     scales [kq][rows] 32-bit words, byte b = block b of that quad of that row.
// One lane's operand of v_mfma_scale_f32_16x16x128_f8f6f4 is one block (16 bytes of codes, one scale
// byte), and the 16 rows that 16 lanes hold have their scale words next to each other.
#pragma once

#include <cstddef>
#include <cstdint>
#include <string>

namespace gpumon_hip {

constexpr int64_t kMxBlock = 32, kMxQuad = 128;
inline int64_t mx_quads(int64_t k) { return (k + kMxQuad - 1) / kMxQuad; }
// bytes of codes and of scales
inline int64_t mx_codes_bytes(int64_t rows, int64_t k) { return rows * mx_quads(k) * 64; }
inline int64_t mx_scales_bytes(int64_t rows, int64_t k) { return rows * mx_quads(k) * 4; }

// All launches: dtype bf16 | f16 | f32; strides in elements; codes 16-byte, scales 4-byte aligned.
// They throw std::invalid_argument before anything is launched, keep the calling thread's current
// device, and need no synchronisation: they can be recorded into a graph.

// x [rows, k], element (r, c) at x[r * stride + c]. by_column: the result has x's columns as its rows,
// with blocks of 32 consecutive rows of x (k rows of length `rows`).
void launch_mx_quantize(int dev, const void* x, const std::string& dtype, int64_t rows, int64_t k, int64_t stride,
                        bool by_column, void* codes, void* scales, void* stream);
// Both results of the two directions from one reading of x.
void launch_mx_quantize_both(int dev, const void* x, const std::string& dtype, int64_t rows, int64_t k, int64_t stride,
                             void* row_codes, void* row_scales, void* col_codes, void* col_scales, void* stream);
// out [rows, k], element (r, c) at out[r * stride + c].
void launch_mx_dequantize(int dev, const void* codes, const void* scales, int64_t rows, int64_t k, void* out,
                          const std::string& dtype, int64_t stride, void* stream);
// c [m, n] = a [m, k] b [n, k]^T, sums in 32 bits, rounded once. workspace: mx_product_workspace bytes.
size_t mx_product_workspace(int dev, int64_t m, int64_t n, int64_t k);
void launch_mx_product(int dev, const void* a_codes, const void* a_scales, const void* b_codes, const void* b_scales,
                       int64_t m, int64_t n, int64_t k, void* c, const std::string& dtype, int64_t stride,
                       void* workspace, size_t workspace_bytes, void* stream);
// y [m, n] = Q(x) w^T: x [m, k] in `dtype`, quantised here; y has the same type.
size_t mx_linear_workspace(int dev, int64_t m, int64_t n, int64_t k);
void launch_mx_linear(int dev, const void* x, const std::string& dtype, int64_t x_stride, const void* w_codes,
                      const void* w_scales, int64_t m, int64_t n, int64_t k, void* y, int64_t y_stride,
                      void* workspace, size_t workspace_bytes, void* stream);

}  // namespace gpumon_hip
