// pybind11 bindings: gpumon._hip (gfx950 kernels: K1 probe, K2 synthetic load).
// Pointers/streams are passed as integers (torch tensor .data_ptr(), torch.cuda stream handle) so
// the kernels can be checked against PyTorch fp32 references on the same tensors.
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include "../hip/hip_api.h"
#include "../hip/mx.h"
#include "../hip/mx_load.h"

namespace py = pybind11;
using namespace gpumon_hip;

static void* P(uintptr_t x) { return reinterpret_cast<void*>(x); }

static py::dict load_stats(const LoadStats& s) {
  py::dict d;
  d["launches"] = s.launches;
  d["busy_s"] = s.busy_s;
  d["flops"] = s.flops;
  d["bytes"] = s.bytes;
  d["mfma_s"] = s.mfma_s;
  d["hbm_s"] = s.hbm_s;
  d["wall_s"] = s.wall_s;
  d["tflops"] = s.mfma_s > 0 ? s.flops / s.mfma_s / 1e12 : 0.0;  // rate while MFMA batches ran
  d["tbps"] = s.hbm_s > 0 ? s.bytes / s.hbm_s / 1e12 : 0.0;      // rate while HBM batches ran
  d["tflops_wall"] = s.wall_s > 0 ? s.flops / s.wall_s / 1e12 : 0.0;  // averaged over wall time
  d["tbps_wall"] = s.wall_s > 0 ? s.bytes / s.wall_s / 1e12 : 0.0;
  return d;
}

PYBIND11_MODULE(_hip, m) {
  m.doc() = "gpumon gfx950 HIP kernels (probe ring buffer + synthetic MFMA/HBM load)";
  m.def("device_count", &device_count);
  m.def("device_arch", &device_arch);
  m.def("device_cu_count", &device_cu_count);
  m.def("device_pci_bus_id", &device_pci_bus_id);

  m.def("mfma_tile", [](int dev, uintptr_t a, uintptr_t b, uintptr_t c, int iters, uintptr_t stream) {
    launch_mfma_tile(dev, P(a), P(b), static_cast<float*>(P(c)), iters, P(stream));
  }, py::arg("dev"), py::arg("a"), py::arg("b"), py::arg("c"), py::arg("iters"), py::arg("stream") = 0);
  m.def("mfma_burn", [](int dev, uintptr_t a, uintptr_t b, uintptr_t out, int blocks, int iters, uintptr_t stream,
                        int shape) {
    launch_mfma_burn(dev, P(a), P(b), static_cast<float*>(P(out)), blocks, iters, P(stream), shape);
  }, py::arg("dev"), py::arg("a"), py::arg("b"), py::arg("out"), py::arg("blocks"), py::arg("iters"),
     py::arg("stream") = 0, py::arg("shape") = 32);
  m.def("mfma_burn_dtype", [](int dev, const std::string& dtype, uintptr_t out, int blocks, int iters,
                              uintptr_t stream) {
    return launch_mfma_burn_dtype(dev, dtype, static_cast<float*>(P(out)), blocks, iters, P(stream));
  }, py::arg("dev"), py::arg("dtype"), py::arg("out"), py::arg("blocks"), py::arg("iters"), py::arg("stream") = 0,
     "MFMA burn of one matrix path (f16|fp8|f32|f64|i8|mxfp8|mxfp4); returns FLOP per launch");
  m.def("stream_copy", [](int dev, uintptr_t src, uintptr_t dst, size_t n16, int blocks, uintptr_t stream,
                          int unroll, int policy, bool span) {
    launch_stream_copy(dev, P(src), P(dst), n16, blocks, P(stream), unroll, policy, span);
  }, py::arg("dev"), py::arg("src"), py::arg("dst"), py::arg("n16"), py::arg("blocks") = 4096,
     py::arg("stream") = 0, py::arg("unroll") = 4, py::arg("policy") = 0, py::arg("span") = false);
  m.def("stream_triad", [](int dev, uintptr_t a, uintptr_t b, uintptr_t c, float s, size_t n, int blocks,
                           uintptr_t stream) {
    launch_stream_triad(dev, static_cast<const float*>(P(a)), static_cast<const float*>(P(b)),
                        static_cast<float*>(P(c)), s, n, blocks, P(stream));
  }, py::arg("dev"), py::arg("a"), py::arg("b"), py::arg("c"), py::arg("s"), py::arg("n"),
     py::arg("blocks") = 4096, py::arg("stream") = 0);

  // MXFP4 operators (mx.h; on tensors: gpumon.ops.mx)
  m.def("mx_quantize", [](int dev, uintptr_t x, const std::string& dtype, int64_t rows, int64_t k, int64_t stride,
                          bool by_column, uintptr_t codes, uintptr_t scales, uintptr_t stream) {
    launch_mx_quantize(dev, P(x), dtype, rows, k, stride, by_column, P(codes), P(scales), P(stream));
  }, py::arg("dev"), py::arg("x"), py::arg("dtype"), py::arg("rows"), py::arg("k"), py::arg("stride"),
     py::arg("by_column"), py::arg("codes"), py::arg("scales"), py::arg("stream") = 0);
  m.def("mx_quantize_both", [](int dev, uintptr_t x, const std::string& dtype, int64_t rows, int64_t k, int64_t stride,
                               uintptr_t row_codes, uintptr_t row_scales, uintptr_t col_codes, uintptr_t col_scales,
                               uintptr_t stream) {
    launch_mx_quantize_both(dev, P(x), dtype, rows, k, stride, P(row_codes), P(row_scales), P(col_codes),
                            P(col_scales), P(stream));
  }, py::arg("dev"), py::arg("x"), py::arg("dtype"), py::arg("rows"), py::arg("k"), py::arg("stride"),
     py::arg("row_codes"), py::arg("row_scales"), py::arg("col_codes"), py::arg("col_scales"), py::arg("stream") = 0);
  m.def("mx_dequantize", [](int dev, uintptr_t codes, uintptr_t scales, int64_t rows, int64_t k, uintptr_t out,
                            const std::string& dtype, int64_t stride, uintptr_t stream) {
    launch_mx_dequantize(dev, P(codes), P(scales), rows, k, P(out), dtype, stride, P(stream));
  }, py::arg("dev"), py::arg("codes"), py::arg("scales"), py::arg("rows"), py::arg("k"), py::arg("out"),
     py::arg("dtype"), py::arg("stride"), py::arg("stream") = 0);
  m.def("mx_product_workspace", &mx_product_workspace, py::arg("m"), py::arg("n"), py::arg("k"));
  m.def("mx_product_kernel", &mx_product_kernel, py::arg("m"), py::arg("n"), py::arg("k"));
  m.def("mx_product", [](int dev, uintptr_t a_codes, uintptr_t a_scales, uintptr_t b_codes, uintptr_t b_scales,
                         int64_t m, int64_t n, int64_t k, uintptr_t c, const std::string& dtype, int64_t stride,
                         uintptr_t workspace, size_t workspace_bytes, uintptr_t stream) {
    launch_mx_product(dev, P(a_codes), P(a_scales), P(b_codes), P(b_scales), m, n, k, P(c), dtype, stride,
                      P(workspace), workspace_bytes, P(stream));
  }, py::arg("dev"), py::arg("a_codes"), py::arg("a_scales"), py::arg("b_codes"), py::arg("b_scales"), py::arg("m"),
     py::arg("n"), py::arg("k"), py::arg("c"), py::arg("dtype"), py::arg("stride"), py::arg("workspace") = 0,
     py::arg("workspace_bytes") = 0, py::arg("stream") = 0);
  m.def("mx_linear_workspace", &mx_linear_workspace, py::arg("m"), py::arg("n"), py::arg("k"), py::arg("dtype"));
  m.def("mx_linear_kernel", &mx_linear_kernel, py::arg("m"), py::arg("n"), py::arg("k"), py::arg("dtype"));
  m.def("mx_linear", [](int dev, uintptr_t x, const std::string& dtype, int64_t x_stride, uintptr_t w_codes,
                        uintptr_t w_scales, int64_t m, int64_t n, int64_t k, uintptr_t y, int64_t y_stride,
                        uintptr_t workspace, size_t workspace_bytes, uintptr_t stream) {
    launch_mx_linear(dev, P(x), dtype, x_stride, P(w_codes), P(w_scales), m, n, k, P(y), y_stride, P(workspace),
                     workspace_bytes, P(stream));
  }, py::arg("dev"), py::arg("x"), py::arg("dtype"), py::arg("x_stride"), py::arg("w_codes"), py::arg("w_scales"),
     py::arg("m"), py::arg("n"), py::arg("k"), py::arg("y"), py::arg("y_stride"), py::arg("workspace") = 0,
     py::arg("workspace_bytes") = 0, py::arg("stream") = 0);

  m.def("mx_linear_train_saved", &mx_linear_train_saved, py::arg("m"), py::arg("n"), py::arg("k"));
  m.def("mx_linear_train_workspace", &mx_linear_train_workspace, py::arg("m"), py::arg("n"), py::arg("k"));
  m.def("mx_linear_train", [](int dev, uintptr_t x, const std::string& dtype, int64_t x_stride, uintptr_t w,
                              const std::string& w_dtype, int64_t w_stride, int64_t m, int64_t n, int64_t k,
                              uintptr_t y, int64_t y_stride, uintptr_t saved, size_t saved_bytes, uintptr_t workspace,
                              size_t workspace_bytes, uintptr_t stream) {
    launch_mx_linear_train(dev, P(x), dtype, x_stride, P(w), w_dtype, w_stride, m, n, k, P(y), y_stride, P(saved),
                           saved_bytes, P(workspace), workspace_bytes, P(stream));
  }, py::arg("dev"), py::arg("x"), py::arg("dtype"), py::arg("x_stride"), py::arg("w"), py::arg("w_dtype"),
     py::arg("w_stride"), py::arg("m"), py::arg("n"), py::arg("k"), py::arg("y"), py::arg("y_stride"),
     py::arg("saved"), py::arg("saved_bytes"), py::arg("workspace"), py::arg("workspace_bytes"), py::arg("stream") = 0);
  m.def("mx_linear_grad_workspace", &mx_linear_grad_workspace, py::arg("m"), py::arg("n"), py::arg("k"));
  m.def("mx_linear_grad_kernel", &mx_linear_grad_kernel, py::arg("m"), py::arg("n"), py::arg("k"));
  m.def("mx_linear_grad", [](int dev, uintptr_t dy, const std::string& dtype, int64_t dy_stride, uintptr_t saved,
                             int64_t m, int64_t n, int64_t k, uintptr_t dx, int64_t dx_stride, uintptr_t dw,
                             const std::string& w_dtype, int64_t dw_stride, uintptr_t workspace, size_t workspace_bytes,
                             uintptr_t stream) {
    launch_mx_linear_grad(dev, P(dy), dtype, dy_stride, P(saved), m, n, k, P(dx), dx_stride, P(dw), w_dtype, dw_stride,
                          P(workspace), workspace_bytes, P(stream));
  }, py::arg("dev"), py::arg("dy"), py::arg("dtype"), py::arg("dy_stride"), py::arg("saved"), py::arg("m"),
     py::arg("n"), py::arg("k"), py::arg("dx"), py::arg("dx_stride"), py::arg("dw"), py::arg("w_dtype"),
     py::arg("dw_stride"), py::arg("workspace"), py::arg("workspace_bytes"), py::arg("stream") = 0);

  py::class_<LoadGen>(m, "LoadGen")
      .def(py::init([](int dev, std::string kind, double duty, size_t hbm_bytes, int mfma_iters, int shape,
                       std::string dtype, double period_s) {
             auto g = std::make_unique<LoadGen>(dev, std::move(kind), duty, hbm_bytes, mfma_iters);
             g->set_mfma_shape(shape);
             g->set_mfma_dtype(std::move(dtype));
             g->set_period(period_s);
             return g;
           }),
           py::arg("dev"), py::arg("kind") = "mixed", py::arg("duty") = 1.0, py::arg("hbm_bytes") = size_t(1) << 30,
           py::arg("mfma_iters") = 8192, py::arg("mfma_shape") = 32, py::arg("mfma_dtype") = "bf16",
           py::arg("period_s") = 0.0)
      .def("start", [](LoadGen& g) {
        py::gil_scoped_release nogil;
        g.start();
      })
      .def("stop", [](LoadGen& g) {
        py::gil_scoped_release nogil;
        g.stop();
      })
      .def_property_readonly("running", &LoadGen::running)
      .def("stats", [](LoadGen& g) {
        return load_stats(g.stats());
      });

  py::class_<MxLoad>(m, "MxLoad")
      .def(py::init<int, int64_t, int64_t, int64_t, double, double>(), py::arg("dev"), py::arg("rows") = 4096,
           py::arg("n") = 8192, py::arg("k") = 8192, py::arg("duty") = 1.0, py::arg("period_s") = 0.0)
      .def("start", [](MxLoad& g) {
        py::gil_scoped_release nogil;
        g.start();
      })
      .def("stop", [](MxLoad& g) {
        py::gil_scoped_release nogil;
        g.stop();
      })
      .def_property_readonly("running", &MxLoad::running)
      .def("stats", [](MxLoad& g) { return load_stats(g.stats()); });

  py::class_<XgmiLoad>(m, "XgmiLoad")
      .def(py::init<int, int, size_t, std::string, int>(), py::arg("src"), py::arg("dst"),
           py::arg("nbytes") = size_t(256) << 20, py::arg("method") = "kernel", py::arg("blocks") = 512)
      .def("start", [](XgmiLoad& g) {
        py::gil_scoped_release nogil;
        g.start();
      })
      .def("stop", [](XgmiLoad& g) {
        py::gil_scoped_release nogil;
        g.stop();
      })
      .def_property_readonly("running", &XgmiLoad::running)
      .def("stats", [](XgmiLoad& g) {
        XgmiStats s = g.stats();
        py::dict d;
        d["copies"] = s.copies;
        d["bytes"] = s.bytes;
        d["busy_s"] = s.busy_s;
        d["wall_s"] = s.wall_s;
        d["GBps"] = s.busy_s > 0 ? s.bytes / s.busy_s / 1e9 : 0.0;       // while copying
        d["GBps_wall"] = s.wall_s > 0 ? s.bytes / s.wall_s / 1e9 : 0.0;  // averaged over wall time
        return d;
      });

  py::class_<PcieLoad>(m, "PcieLoad")
      .def(py::init<int, size_t, std::string, double>(), py::arg("dev"), py::arg("nbytes") = size_t(256) << 20,
           py::arg("direction") = "both", py::arg("duty") = 1.0)
      .def("start", [](PcieLoad& g) {
        py::gil_scoped_release nogil;
        g.start();
      })
      .def("stop", [](PcieLoad& g) {
        py::gil_scoped_release nogil;
        g.stop();
      })
      .def_property_readonly("running", &PcieLoad::running)
      .def("stats", [](PcieLoad& g) {
        PcieStats s = g.stats();
        py::dict d;
        d["copies"] = s.copies;
        d["h2d_bytes"] = s.h2d_bytes;
        d["d2h_bytes"] = s.d2h_bytes;
        d["bytes"] = s.h2d_bytes + s.d2h_bytes;
        d["busy_s"] = s.busy_s;
        d["wall_s"] = s.wall_s;
        d["GBps_wall"] = s.wall_s > 0 ? (s.h2d_bytes + s.d2h_bytes) / s.wall_s / 1e9 : 0.0;  // both directions
        return d;
      });

  py::class_<Probe>(m, "Probe")
      .def(py::init<int, int, int, int>(), py::arg("dev"), py::arg("blocks") = 1024, py::arg("slots") = 4,
           py::arg("spin_ticks") = 200)
      .def("launch", &Probe::launch)
      .def_property_readonly("blocks", &Probe::blocks)
      .def("poll", [](Probe& p, int slot, double timeout_s) -> py::object {
        ProbeResult r;
        bool ok;
        {
          py::gil_scoped_release nogil;
          ok = timeout_s > 0 ? p.wait(slot, timeout_s, &r) : p.poll(slot, &r);
        }
        if (!ok) return py::none();
        py::dict d;
        d["seq"] = r.seq;
        d["blocks"] = r.blocks;
        d["arrived"] = r.arrived;
        d["host_latency_s"] = (r.host_done_ns - r.host_launch_ns) * 1e-9;
        d["gpu_span_s"] = r.gpu_span_ticks * 1e-8;
        d["xcc_blocks"] = r.xcc_blocks;
        d["xcc_clock_mhz"] = r.xcc_clock_mhz;
        d["unique_cus"] = r.unique_cus;
        d["xcc_wave_slot"] = r.xcc_wave_slot;
        d["wave_slot_mean"] = r.wave_slot_mean;
        d["stale_records"] = r.stale_records;
        py::list recs;
        for (const auto& x : r.records)
          recs.append(py::make_tuple(x.xcc_id, x.hw_id, x.t0_real, x.t1_real, x.c0, x.c1, x.seq, x.block));
        d["records"] = recs;
        return d;
      }, py::arg("slot"), py::arg("timeout_s") = 0.0);
}
