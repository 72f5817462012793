// MXFP4 operators: quantisation, product and linear layer (mx_quant.hip, mx_product.hip).
//
// Format. A matrix of `rows` x `k` is held in blocks of 32 consecutive elements of a row: 4 bits an
// element (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) and one scale byte a block (e8m0:
// 2^(byte - 127); 255: the block stands for NaN). With amax the block's largest magnitude,
//     E = clamp(floor(log2 amax) - 2, -127, 125)   (amax = 0: -127),   byte = E + 127,
//     q_i = x_i / 2^E rounded to the grid, halves to the even code, beyond 6 to 6;
// a NaN or an infinity in the block: byte 255. Dividing by 2^E is exact, so every code is determined.
//
// Layout. Rows are filled up to blocks of 16 and k with zeros to quads of 128 elements (4 scale blocks):
//     codes  [row block][quad][4 blocks][16 rows][16 bytes], the even element in the low nibble;
//     scales [row block][group of 4 quads][4 blocks][16 rows][4 quads] bytes, zeros past the last quad.
// A lane's operand of v_mfma_scale_f32_16x16x128_f8f6f4 is one block of one row (lane l: row l & 15,
// block l >> 4), so a wave's operand is one "chunk" of 1 KiB in lane order, and the scale words of
// four such steps are 256 bytes in lane order, the instruction picking the step's byte. Memory, LDS
// and registers hold the same order: every transfer is contiguous, without shuffles and with few
// bank conflicts (3 % of the LDS cycles of an 8192^3 product).
#pragma once

#include <cstddef>
#include <cstdint>
#include <string>

namespace gpumon_hip {

inline int64_t mx_quads(int64_t k) { return (k + 127) / 128; }
inline int64_t mx_groups(int64_t k) { return (k + 511) / 512; }
inline int64_t mx_row_blocks(int64_t rows) { return (rows + 15) / 16; }
// bytes of codes and of scales
inline int64_t mx_codes_bytes(int64_t rows, int64_t k) { return mx_row_blocks(rows) * mx_quads(k) * 1024; }
inline int64_t mx_scales_bytes(int64_t rows, int64_t k) { return mx_row_blocks(rows) * mx_groups(k) * 256; }
// Limits of the kernels' indexes and grids: 2^24 pieces of 16 rows x 512 elements (more than fits the
// card in 16 bits an element) and 2^28 elements along a row (a row block's offsets stay within 32
// bits); a product also has at most 2^28 pieces of 16 x 16 results, and quantising down the columns fewer
// than 2^23 tiles of 32 x 512 in a launch.
inline bool mx_fits(int64_t rows, int64_t k) {
  return rows < (1ll << 28) && k <= (1ll << 28) && mx_row_blocks(rows) * mx_groups(k) < (1ll << 24);
}

// All launches: dtype bf16 | f16 | f32; strides in elements; codes and scales 16-byte aligned.
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
size_t mx_product_workspace(int64_t m, int64_t n, int64_t k);
// The kernel that these sizes take: a tile's "256x256" to "64x64", "64x64/3" with k in three parts, or "few16" to
// "few64x2" for few rows.
std::string mx_product_kernel(int64_t m, int64_t n, int64_t k);
void launch_mx_product(int dev, const void* a_codes, const void* a_scales, const void* b_codes, const void* b_scales,
                       int64_t m, int64_t n, int64_t k, void* c, const std::string& dtype, int64_t stride,
                       void* workspace, size_t workspace_bytes, void* stream);
// y [m, n] = Q(x) w^T: x [m, k] in `dtype`, quantised here; y has the same type.
size_t mx_linear_workspace(int64_t m, int64_t n, int64_t k, const std::string& dtype);
// The product's kernel as above, or "way1" to "way8x2" where it quantises x on the way.
std::string mx_linear_kernel(int64_t m, int64_t n, int64_t k, const std::string& dtype);
void launch_mx_linear(int dev, const void* x, const std::string& dtype, int64_t x_stride, const void* w_codes,
                      const void* w_scales, int64_t m, int64_t n, int64_t k, void* y, int64_t y_stride,
                      void* workspace, size_t workspace_bytes, void* stream);


// Training step of a linear layer. Forward: y [m, n] = Q(x) Q(w)^T from x [m, k] and w [n, k], with x and w
// quantised down their columns too, into `saved`. Backward: dx [m, k] = Q(dy) Q0(w), dw [n, k] =
// Q0(dy)^T Q0(x), Q0 in blocks down the columns; dx or dw may be null. y and dx have x's type, dw w's.
size_t mx_linear_train_saved(int64_t m, int64_t n, int64_t k);
size_t mx_linear_train_workspace(int64_t m, int64_t n, int64_t k);
void launch_mx_linear_train(int dev, const void* x, const std::string& dtype, int64_t x_stride, const void* w,
                            const std::string& w_dtype, int64_t w_stride, int64_t m, int64_t n, int64_t k, void* y,
                            int64_t y_stride, void* saved, size_t saved_bytes, void* workspace, size_t workspace_bytes,
                            void* stream);
// A gradient has the same bits whether the other is asked for or not.
size_t mx_linear_grad_workspace(int64_t m, int64_t n, int64_t k);
// The tile that both gradients of one type take in one launch, or "" where each has its own (mx_product_kernel).
std::string mx_linear_grad_kernel(int64_t m, int64_t n, int64_t k);
void launch_mx_linear_grad(int dev, const void* dy, const std::string& dtype, int64_t dy_stride, const void* saved,
                           int64_t m, int64_t n, int64_t k, void* dx, int64_t dx_stride, void* dw,
                           const std::string& w_dtype, int64_t dw_stride, void* workspace, size_t workspace_bytes,
                           void* stream);

}  // namespace gpumon_hip
