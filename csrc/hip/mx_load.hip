#include "mx_load.h"

#include <algorithm>
#include <chrono>

#include "mx.h"
#include "mx_common.h"

namespace gpumon_hip {

namespace {

int64_t now_ns() {
  return std::chrono::duration_cast<std::chrono::nanoseconds>(std::chrono::steady_clock::now().time_since_epoch()).count();
}

// bf16 values near a normal distribution: the sum of four uniform ones from a hash of the index (the published
// 64-bit mixer splitmix64).
__global__ void __launch_bounds__(256) random_kernel(__bf16* x, size_t n, uint32_t seed) {
  for (size_t i = blockIdx.x * size_t{256} + threadIdx.x; i < n; i += size_t{256} * gridDim.x) {
    uint64_t h = (i + 1) * 0x9e3779b97f4a7c15ull + seed;
    h = (h ^ (h >> 30)) * 0xbf58476d1ce4e5b9ull;
    h = (h ^ (h >> 27)) * 0x94d049bb133111ebull;
    h ^= h >> 31;
    const int sum = static_cast<int>(h & 0xffff) + static_cast<int>(h >> 16 & 0xffff) + static_cast<int>(h >> 32 & 0xffff) +
                    static_cast<int>(h >> 48) - 2 * 0xffff;
    x[i] = static_cast<__bf16>(static_cast<float>(sum) * (1.732f / 65536.f));
  }
}

constexpr int64_t kWeightBytes = int64_t{512} << 20;

}  // namespace

MxLoad::MxLoad(int dev, int64_t rows, int64_t n, int64_t k, double duty, double period_s)
    : dev_(dev), rows_(rows), n_(n), k_(k), duty_(std::clamp(duty, 0.01, 1.0)), period_s_(period_s) {
  mx::require(rows >= 1 && n >= 1 && k >= 1, "MxLoad: rows, n and k must be at least 1");
  workspace_bytes_ = mx_linear_workspace(rows, n, k, "bf16");  // checks the sizes' limits
}

MxLoad::~MxLoad() { stop(); }

void MxLoad::start() {
  if (running_) return;
  stop();  // a thread that ended by an error is still to be joined
  failed_ = false;
  check(hipSetDevice(dev_), "hipSetDevice");
  try {
    hipStream_t s;
    check(hipStreamCreateWithFlags(&s, hipStreamNonBlocking), "hipStreamCreate");
    stream_ = s;
    const size_t scales_at = static_cast<size_t>(mx_codes_bytes(n_, k_));
    layer_bytes_ = scales_at + static_cast<size_t>(mx_scales_bytes(n_, k_));
    layers_ = std::clamp<size_t>((kWeightBytes + layer_bytes_ - 1) / layer_bytes_, 2, 4096);
    check(hipMalloc(reinterpret_cast<void**>(&weights_), layers_ * layer_bytes_), "hipMalloc");
    check(hipMalloc(&x_, static_cast<size_t>(std::max(n_, rows_) * k_) * 2), "hipMalloc");  // the plain weights first
    for (size_t i = 0; i < layers_; ++i) {
      char* w = weights_ + i * layer_bytes_;
      hipLaunchKernelGGL(random_kernel, dim3(4096), dim3(256), 0, s, static_cast<__bf16*>(x_),
                         static_cast<size_t>(n_ * k_), static_cast<uint32_t>(i + 1));
      launch_mx_quantize(dev_, x_, "bf16", n_, k_, k_, false, w, w + scales_at, s);
    }
    hipLaunchKernelGGL(random_kernel, dim3(4096), dim3(256), 0, s, static_cast<__bf16*>(x_), static_cast<size_t>(rows_ * k_), 0u);
    check(hipMalloc(&y_, static_cast<size_t>(rows_ * n_) * 2), "hipMalloc");
    if (workspace_bytes_) check(hipMalloc(&workspace_, workspace_bytes_), "hipMalloc");
    check(hipGetLastError(), "random_kernel");
    check(hipStreamSynchronize(s), "hipStreamSynchronize");
  } catch (...) {
    release();
    throw;
  }
  running_ = true;
  t_start_ns_ = now_ns();
  th_ = std::thread([this] { loop(); });
}

void MxLoad::loop() {
  try {
    check(hipSetDevice(dev_), "hipSetDevice");
    auto s = static_cast<hipStream_t>(stream_);
    hipEvent_t e0, e1;
    check(hipEventCreate(&e0), "hipEventCreate");
    check(hipEventCreate(&e1), "hipEventCreate");
    const size_t scales_at = static_cast<size_t>(mx_codes_bytes(n_, k_));
    // a batch of a millisecond or so, at least four layers, so that the host's wait between batches is small
    const double us = std::max(2.0 * rows_ * n_ * k_ / 4e9, n_ * k_ * 0.53 / 5e6);
    const int batch = static_cast<int>(std::clamp(2000.0 / us, 4.0, 400.0));
    size_t next = 0;
    while (running_) {
      check(hipEventRecord(e0, s), "hipEventRecord");
      for (int i = 0; i < batch; ++i) {
        const char* w = weights_ + next * layer_bytes_;
        next = (next + 1) % layers_;
        launch_mx_linear(dev_, x_, "bf16", k_, w, w + scales_at, rows_, n_, k_, y_, n_, workspace_, workspace_bytes_, s);
      }
      check(hipEventRecord(e1, s), "hipEventRecord");
      check(hipEventSynchronize(e1), "hipEventSynchronize");
      float ms = 0;
      check(hipEventElapsedTime(&ms, e0, e1), "hipEventElapsedTime");
      busy_ns_ += static_cast<uint64_t>(ms * 1e6);
      launches_ += batch;
      if (duty_ < 0.999) {
        // busy until duty * period into the period, then idle to its end; without a period an idle gap a batch
        int64_t until = now_ns() + static_cast<int64_t>(ms * 1e6 * (1.0 / duty_ - 1.0));
        if (period_s_ > 0) {
          const auto per = static_cast<int64_t>(period_s_ * 1e9);
          const int64_t phase = (now_ns() - t_start_ns_) % per;
          until = phase >= static_cast<int64_t>(duty_ * per) ? now_ns() + per - phase : 0;
        }
        while (running_ && now_ns() < until) std::this_thread::sleep_for(std::chrono::microseconds(500));
      }
    }
    (void)hipEventDestroy(e0);
    (void)hipEventDestroy(e1);
  } catch (const std::exception& e) {
    err_ = e.what();
    failed_ = true;
    running_ = false;
  }
}

void MxLoad::release() {
  (void)hipSetDevice(dev_);
  if (stream_) {
    (void)hipStreamSynchronize(static_cast<hipStream_t>(stream_));
    (void)hipStreamDestroy(static_cast<hipStream_t>(stream_));
  }
  if (weights_) (void)hipFree(weights_);
  weights_ = nullptr;
  for (void** p : {&x_, &y_, &workspace_}) {
    if (*p) (void)hipFree(*p);
    *p = nullptr;
  }
  stream_ = nullptr;
}

void MxLoad::stop() {
  running_ = false;
  if (th_.joinable()) th_.join();
  release();
}

LoadStats MxLoad::stats() const {
  if (failed_) throw std::runtime_error("MxLoad failed: " + err_);
  LoadStats s;
  s.launches = launches_;
  s.busy_s = s.mfma_s = s.hbm_s = busy_ns_ * 1e-9;
  const double layers = static_cast<double>(s.launches);
  s.flops = layers * 2.0 * rows_ * n_ * k_;
  s.bytes = layers * (2.0 * rows_ * k_ + 17.0 / 32.0 * n_ * k_ + 2.0 * rows_ * n_);
  s.wall_s = t_start_ns_ ? (now_ns() - t_start_ns_) * 1e-9 : 0.0;
  return s;
}

}  // namespace gpumon_hip
