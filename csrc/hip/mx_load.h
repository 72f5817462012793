// MXFP4 linear layers as a background load (kind "mxlinear"): quantised data, memory traffic and matrix
// instructions together, as a node that serves in 4 bits runs them.
#pragma once

#include <atomic>
#include <cstdint>
#include <string>
#include <thread>

#include "hip_api.h"

namespace gpumon_hip {

class MxLoad {
 public:
  // y [rows, n] = Q(x) w^T back to back, x [rows, k] bf16 of random values. The layers' quantised weights
  // come to at least 512 MiB (or 4096 layers), taken in turn, so that with few rows (decode) they come
  // from HBM, not from a cache. duty / period_s as in LoadGen.
  MxLoad(int dev, int64_t rows, int64_t n, int64_t k, double duty, double period_s);
  ~MxLoad();
  void start();
  void stop();
  // flops: 2 rows n k a layer (the padding of tiles not counted); bytes: x, the layer's weights and y once
  // each; both over the same GPU time, mfma_s = hbm_s = busy_s.
  LoadStats stats() const;
  bool running() const { return running_; }

 private:
  void loop();
  void release();
  int dev_;
  int64_t rows_, n_, k_;
  double duty_, period_s_;
  char* weights_ = nullptr;  // layers_ times codes, then scales
  size_t layers_ = 0, layer_bytes_ = 0;
  void* stream_ = nullptr;
  void* x_ = nullptr;
  void* y_ = nullptr;
  void* workspace_ = nullptr;
  size_t workspace_bytes_ = 0;
  std::thread th_;
  std::atomic<bool> running_{false};
  int64_t t_start_ns_ = 0;
  std::atomic<uint64_t> launches_{0}, busy_ns_{0};
  std::string err_;  // written before failed_
  std::atomic<bool> failed_{false};
};

}  // namespace gpumon_hip
