// Python bindings of the native runtime (pybind11, no torch headers).
//
// Tensors cross the boundary as raw device addresses (tensor.data_ptr()) and streams as
// hipStream_t handles (torch.cuda.current_stream().cuda_stream); the Python wrappers in
// ops/native.py validate dtype / shape / contiguity before calling in.  Memory is owned
// by the torch caching allocator, the native side never frees or allocates tensors.
#include <tuple>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <stdexcept>
#include <string>
#include <vector>

#include "dml_comm.h"
#include "dml_engine.h"
#include "dml_kernels.h"
#include "dml_newton_schulz.h"

namespace py = pybind11;
namespace dml {
void launch_pollers(int blocks, long long ticks, const unsigned* flag, hipStream_t stream);
}
using namespace dml;

namespace {

template <typename T>
T* ptr(uintptr_t p) { return reinterpret_cast<T*>(p); }
hipStream_t st(uintptr_t s) { return reinterpret_cast<hipStream_t>(s); }

ConvShape shape(int batch, int hw, int cin, int cout) {
    ConvShape s;
    s.batch = batch; s.hw = hw; s.cin = cin; s.cout = cout;
    return s;
}

}  // namespace

// hash of the source tree this library was built from (generated by build.py at link time)
extern "C" const char dml_build_id[];

PYBIND11_MODULE(_C, m) {
    m.doc() = "MI355X-native kernels, training engine and RCCL communicator";
    m.attr("build_id") = std::string(dml_build_id);

    // ------------------------------------------------------------------ kernels
    m.def("conv3x3_igemm", [](uintptr_t x, uintptr_t w, uintptr_t y, uintptr_t bias, uintptr_t mask,
                              uintptr_t ws, size_t ws_elems, int batch, int hw, int cin, int cout,
                              int epi, uintptr_t stream, int bm, int bn, int splits, int pm,
                              int waves, uintptr_t stats) {
        const int force[5] = {bm, bn, splits, pm, waves};
        conv3x3_igemm(ptr<const bf16_raw>(x), ptr<const bf16_raw>(w), ptr<bf16_raw>(y),
                      ptr<const float>(bias), ptr<const bf16_raw>(mask), ptr<float>(ws), ws_elems,
                      shape(batch, hw, cin, cout), (ConvEpilogue)epi, st(stream),
                      bm > 0 ? force : nullptr, ptr<float>(stats));
    }, py::arg("x"), py::arg("w"), py::arg("y"), py::arg("bias"), py::arg("mask"), py::arg("ws"),
       py::arg("ws_elems"), py::arg("batch"), py::arg("hw"), py::arg("cin"), py::arg("cout"),
       py::arg("epi"), py::arg("stream"), py::arg("bm") = 0, py::arg("bn") = 0,
       py::arg("splits") = 0, py::arg("pm") = -1, py::arg("waves") = 4, py::arg("stats") = 0);
    // backward-data pass that also leaves the BatchNorm + pool backward sums of the layer whose
    // pooled gradient it writes; returns the number of partial rows (0: the plan cannot)
    m.def("conv3x3_igemm_bn_pool", [](uintptr_t x, uintptr_t w, uintptr_t y, uintptr_t ws,
                                      size_t ws_elems, int batch, int hw, int cin, int cout,
                                      uintptr_t stream, uintptr_t pre, uintptr_t gamma,
                                      uintptr_t beta, uintptr_t mean, uintptr_t rstd,
                                      uintptr_t partials, bool pooled) {
        BnPoolReduce red;
        red.pooled = pooled;
        red.pre = ptr<const bf16_raw>(pre);
        red.gamma = ptr<const float>(gamma); red.beta = ptr<const float>(beta);
        red.mean = ptr<const float>(mean); red.rstd = ptr<const float>(rstd);
        red.partials = ptr<float>(partials);
        BnPartials done;
        conv3x3_igemm(ptr<const bf16_raw>(x), ptr<const bf16_raw>(w), ptr<bf16_raw>(y), nullptr,
                      nullptr, ptr<float>(ws), ws_elems, shape(batch, hw, cin, cout), EPI_NONE,
                      st(stream), nullptr, nullptr, nullptr, &red, &done);
        return done.data ? done.rows : 0;
    }, py::arg("x"), py::arg("w"), py::arg("y"), py::arg("ws"), py::arg("ws_elems"),
       py::arg("batch"), py::arg("hw"), py::arg("cin"), py::arg("cout"), py::arg("stream"),
       py::arg("pre"), py::arg("gamma"), py::arg("beta"), py::arg("mean"), py::arg("rstd"),
       py::arg("partials"), py::arg("pooled") = true);
    m.def("conv3x3_igemm_stats_rows", [](int batch, int hw, int cin, int cout) {
        return conv3x3_igemm_stats_rows(shape(batch, hw, cin, cout));
    });
    m.def("conv1_fprop_stats_rows", &conv1_fprop_stats_rows);
    m.def("conv3x3_igemm_workspace_elems", [](int batch, int hw, int cin, int cout) {
        return conv3x3_igemm_workspace_elems(shape(batch, hw, cin, cout));
    });
    m.def("conv3x3_wgrad", [](uintptr_t x, uintptr_t dy, uintptr_t dw, int batch, int hw, int cin,
                              int cout, uintptr_t stream, int splits, uintptr_t slab) {
        conv3x3_wgrad(ptr<const bf16_raw>(x), ptr<const bf16_raw>(dy), ptr<float>(dw),
                      shape(batch, hw, cin, cout), st(stream), splits, ptr<float>(slab));
    }, py::arg("x"), py::arg("dy"), py::arg("dw"), py::arg("batch"), py::arg("hw"),
       py::arg("cin"), py::arg("cout"), py::arg("stream"), py::arg("splits") = 0,
       py::arg("slab") = 0);
    m.def("conv3x3_wgrad_splits", [](int batch, int hw, int cin, int cout, int target) {
        return conv3x3_wgrad_splits(shape(batch, hw, cin, cout), target);
    }, py::arg("batch"), py::arg("hw"), py::arg("cin"), py::arg("cout"), py::arg("target") = 0);
    m.def("conv3x3_wgrad_max_splits", [](int batch, int hw, int cin, int cout) {
        return conv3x3_wgrad_max_splits(shape(batch, hw, cin, cout));
    });
    m.def("set_wgrad_variant", &set_wgrad_variant);
    m.def("set_wgrad_block_target", &set_wgrad_block_target);
    m.def("set_wgrad_kstep", &set_wgrad_kstep);
    m.def("set_wgrad_waves", &set_wgrad_waves);
    m.def("set_wgrad9_config", &set_wgrad9_config);
    m.def("wgrad_variant", &wgrad_variant);
    m.def("conv3x3_wgrad9_splits", [](int batch, int hw, int cin, int cout, int bco, int force,
                                      int target) {
        const ConvShape s = shape(batch, hw, cin, cout);
        return conv3x3_wgrad9_splits(s, conv3x3_wgrad9_bco(s, bco), force, target);
    }, py::arg("batch"), py::arg("hw"), py::arg("cin"), py::arg("cout"), py::arg("bco") = 0,
       py::arg("force") = 0, py::arg("target") = 0);
    m.def("conv3x3_wgrad9", [](uintptr_t x, uintptr_t dy, uintptr_t dw, int batch, int hw, int cin,
                               int cout, uintptr_t stream, uintptr_t slab, int bco, int splits,
                               int stages) {
        const ConvShape s = shape(batch, hw, cin, cout);
        conv3x3_wgrad9(ptr<const bf16_raw>(x), ptr<const bf16_raw>(dy), ptr<float>(dw), s,
                       st(stream), ptr<float>(slab), conv3x3_wgrad9_bco(s, bco), splits, stages);
    }, py::arg("x"), py::arg("dy"), py::arg("dw"), py::arg("batch"), py::arg("hw"),
       py::arg("cin"), py::arg("cout"), py::arg("stream"), py::arg("slab") = 0,
       py::arg("bco") = 0, py::arg("splits") = 1, py::arg("stages") = 3);
    m.def("sum_slabs_batch", [](uintptr_t src, uintptr_t dst, std::vector<size_t> src_off,
                                std::vector<size_t> dst_off, std::vector<size_t> count,
                                std::vector<int> splits, uintptr_t stream) {
        SlabSumJobs jobs;
        if (src_off.size() > (size_t)SlabSumJobs::kMax || src_off.size() != dst_off.size() ||
            src_off.size() != count.size() || src_off.size() != splits.size())
            throw std::invalid_argument("sum_slabs_batch: bad job lists");
        jobs.n = (int)src_off.size();
        for (int j = 0; j < jobs.n; ++j) {
            jobs.src_off[j] = src_off[j]; jobs.dst_off[j] = dst_off[j];
            jobs.count[j] = count[j]; jobs.splits[j] = splits[j];
        }
        sum_slabs_batch(ptr<const float>(src), ptr<float>(dst), jobs, st(stream));
    });
    m.def("conv1_fprop", [](uintptr_t x, uintptr_t w1, uintptr_t bias, uintptr_t y, int batch,
                            bool relu, uintptr_t stream, uintptr_t stats) {
        conv1_fprop(ptr<const bf16_raw>(x), ptr<const bf16_raw>(w1), ptr<const float>(bias),
                    ptr<bf16_raw>(y), batch, relu, st(stream), ptr<float>(stats));
    }, py::arg("x"), py::arg("w1"), py::arg("bias"), py::arg("y"), py::arg("batch"),
       py::arg("relu"), py::arg("stream"), py::arg("stats") = 0);
    m.def("conv1_wgrad", [](uintptr_t x, uintptr_t dy, uintptr_t dw, uintptr_t db, int batch,
                            uintptr_t ws, uintptr_t stream) {
        conv1_wgrad(ptr<const bf16_raw>(x), ptr<const bf16_raw>(dy), ptr<float>(dw), ptr<float>(db),
                    batch, ptr<float>(ws), st(stream));
    });
    m.def("conv1_wgrad_workspace_elems", &conv1_wgrad_workspace_elems);
    m.def("conv1_wgrad_relu_pool", [](uintptr_t x, uintptr_t act, uintptr_t dyp, uintptr_t dw,
                                      uintptr_t db, int batch, uintptr_t ws, uintptr_t s) {
        conv1_wgrad_relu_pool(ptr<const bf16_raw>(x), ptr<const bf16_raw>(act),
                              ptr<const bf16_raw>(dyp), ptr<float>(dw), ptr<float>(db), batch,
                              ptr<float>(ws), st(s));
    });
    m.def("conv1_wgrad_bn_pool", [](uintptr_t x, uintptr_t pre, uintptr_t dyp, uintptr_t gamma,
                                    uintptr_t beta, uintptr_t mean, uintptr_t rstd, uintptr_t dgamma,
                                    uintptr_t dbeta, uintptr_t dw, int batch, uintptr_t ws,
                                    uintptr_t s) {
        conv1_wgrad_bn_pool(ptr<const bf16_raw>(x), ptr<const bf16_raw>(pre),
                            ptr<const bf16_raw>(dyp), ptr<const float>(gamma), ptr<const float>(beta),
                            ptr<const float>(mean), ptr<const float>(rstd),
                            ptr<const float>(dgamma), ptr<const float>(dbeta), ptr<float>(dw), batch,
                            ptr<float>(ws), st(s));
    });
    m.def("column_reduce_workspace_elems", &bn_workspace_elems);
    m.def("repack_dgrad_weights", [](uintptr_t wf, uintptr_t wd, int cout, int cin, uintptr_t s) {
        repack_dgrad_weights(ptr<const bf16_raw>(wf), ptr<bf16_raw>(wd), cout, cin, st(s));
    });
    m.def("repack_conv1_weights", [](uintptr_t w, uintptr_t w1, uintptr_t s) {
        repack_conv1_weights(ptr<const float>(w), ptr<bf16_raw>(w1), st(s));
    });
    m.def("column_sum", [](uintptr_t x, uintptr_t out, int rows, int cols, uintptr_t ws,
                           uintptr_t s) {
        column_sum(ptr<const bf16_raw>(x), ptr<float>(out), rows, cols, ptr<float>(ws), st(s));
    });
    m.def("maxpool2x2_fwd", [](uintptr_t x, uintptr_t y, int batch, int hw, int c, uintptr_t s) {
        maxpool2x2_fwd(ptr<const bf16_raw>(x), ptr<bf16_raw>(y), batch, hw, c, st(s));
    });
    m.def("maxpool2x2_bwd", [](uintptr_t x, uintptr_t dy, uintptr_t dx, int batch, int hw, int c,
                               bool relu_mask, uintptr_t s) {
        maxpool2x2_bwd(ptr<const bf16_raw>(x), ptr<const bf16_raw>(dy), ptr<bf16_raw>(dx), batch,
                       hw, c, relu_mask, st(s));
    });
    m.def("bn_relu_fwd_train", [](uintptr_t x, uintptr_t y, uintptr_t gamma, uintptr_t beta,
                                  uintptr_t rm, uintptr_t rv, uintptr_t smean, uintptr_t srstd,
                                  uintptr_t ws, int rows, int c, float momentum, float eps,
                                  uintptr_t s) {
        bn_relu_fwd_train(ptr<const bf16_raw>(x), ptr<bf16_raw>(y), ptr<const float>(gamma),
                          ptr<const float>(beta), ptr<float>(rm), ptr<float>(rv), ptr<float>(smean),
                          ptr<float>(srstd), ptr<float>(ws), rows, c, momentum, eps, st(s));
    });
    m.def("bn_relu_fwd_eval", [](uintptr_t x, uintptr_t y, uintptr_t gamma, uintptr_t beta,
                                 uintptr_t rm, uintptr_t rv, int rows, int c, float eps,
                                 uintptr_t s) {
        bn_relu_fwd_eval(ptr<const bf16_raw>(x), ptr<bf16_raw>(y), ptr<const float>(gamma),
                         ptr<const float>(beta), ptr<const float>(rm), ptr<const float>(rv), rows,
                         c, eps, st(s));
    });
    m.def("bn_relu_bwd", [](uintptr_t x, uintptr_t dy, uintptr_t dx, uintptr_t gamma,
                            uintptr_t beta, uintptr_t smean, uintptr_t srstd, uintptr_t dgamma,
                            uintptr_t dbeta, uintptr_t ws, int rows, int c, uintptr_t s,
                            uintptr_t slabs, int splits, size_t stride) {
        bn_relu_bwd(ptr<const bf16_raw>(x), ptr<bf16_raw>(dy), ptr<bf16_raw>(dx),
                    ptr<const float>(gamma), ptr<const float>(beta), ptr<const float>(smean),
                    ptr<const float>(srstd), ptr<float>(dgamma), ptr<float>(dbeta), ptr<float>(ws),
                    rows, c, st(s), SplitSlabs{ptr<const float>(slabs), splits, stride});
    }, py::arg("x"), py::arg("dy"), py::arg("dx"), py::arg("gamma"), py::arg("beta"),
       py::arg("save_mean"), py::arg("save_rstd"), py::arg("dgamma"), py::arg("dbeta"),
       py::arg("ws"), py::arg("rows"), py::arg("c"), py::arg("stream"), py::arg("slabs") = 0,
       py::arg("splits") = 0, py::arg("stride") = 0);
    m.def("bn_relu_pool_fwd_train", [](uintptr_t x, uintptr_t y, uintptr_t gamma, uintptr_t beta,
                                       uintptr_t rmean, uintptr_t rvar, uintptr_t smean,
                                       uintptr_t srstd, uintptr_t ws, int batch, int hw, int c,
                                       float momentum, float eps, uintptr_t s) {
        bn_relu_pool_fwd_train(ptr<const bf16_raw>(x), ptr<bf16_raw>(y), ptr<const float>(gamma),
                               ptr<const float>(beta), ptr<float>(rmean), ptr<float>(rvar),
                               ptr<float>(smean), ptr<float>(srstd), ptr<float>(ws), batch, hw, c,
                               momentum, eps, st(s));
    });
    m.def("bn_relu_pool_fwd_eval", [](uintptr_t x, uintptr_t y, uintptr_t gamma, uintptr_t beta,
                                      uintptr_t rmean, uintptr_t rvar, int batch, int hw, int c,
                                      float eps, uintptr_t s) {
        bn_relu_pool_fwd_eval(ptr<const bf16_raw>(x), ptr<bf16_raw>(y), ptr<const float>(gamma),
                              ptr<const float>(beta), ptr<const float>(rmean),
                              ptr<const float>(rvar), batch, hw, c, eps, st(s));
    });
    m.def("bn_relu_pool_bwd", [](uintptr_t x, uintptr_t dy, uintptr_t dx, uintptr_t gamma,
                                 uintptr_t beta, uintptr_t smean, uintptr_t srstd, uintptr_t dgamma,
                                 uintptr_t dbeta, uintptr_t ws, int batch, int hw, int c,
                                 uintptr_t s, uintptr_t slabs, int splits, size_t stride) {
        bn_relu_pool_bwd(ptr<const bf16_raw>(x), ptr<bf16_raw>(dy), ptr<bf16_raw>(dx),
                         ptr<const float>(gamma), ptr<const float>(beta), ptr<const float>(smean),
                         ptr<const float>(srstd), ptr<float>(dgamma), ptr<float>(dbeta),
                         ptr<float>(ws), batch, hw, c, st(s),
                         SplitSlabs{ptr<const float>(slabs), splits, stride});
    }, py::arg("x"), py::arg("dy"), py::arg("dx"), py::arg("gamma"), py::arg("beta"),
       py::arg("save_mean"), py::arg("save_rstd"), py::arg("dgamma"), py::arg("dbeta"),
       py::arg("ws"), py::arg("batch"), py::arg("hw"), py::arg("c"), py::arg("stream"),
       py::arg("slabs") = 0, py::arg("splits") = 0, py::arg("stride") = 0);
    m.def("conv_tall_tiles", &conv_tall_tiles);
    m.def("set_conv_tall_tiles", &set_conv_tall_tiles);
    m.def("conv_tall_max_rows", &conv_tall_max_rows);
    m.def("set_conv_tall_max_rows", &set_conv_tall_max_rows);
    m.def("launch_pollers", [](int blocks, long long ticks, uintptr_t flag, uintptr_t s) {
        launch_pollers(blocks, ticks, (const unsigned*)flag, (hipStream_t)s);
    });
    m.def("streams_run_concurrently", [](uintptr_t busy, uintptr_t candidate) {
        return streams_run_concurrently((hipStream_t)busy, (hipStream_t)candidate);
    });
    m.def("fc_train", [](uintptr_t x, uintptr_t w, uintptr_t b, uintptr_t target, uintptr_t logits,
                         uintptr_t loss, uintptr_t correct, uintptr_t dx, uintptr_t dw, uintptr_t db,
                         uintptr_t ws, int batch, int in_f, int out_f, uintptr_t s) {
        fc_train(ptr<const bf16_raw>(x), ptr<const float>(w), ptr<const float>(b),
                 ptr<const int64_t>(target), ptr<float>(logits), ptr<float>(loss),
                 ptr<int32_t>(correct), ptr<bf16_raw>(dx), ptr<float>(dw), ptr<float>(db),
                 ptr<float>(ws), batch, in_f, out_f, st(s));
    });
    m.def("fc_train_workspace_elems", &fc_train_workspace_elems);
    m.def("linear_fwd", [](uintptr_t x, uintptr_t w, uintptr_t b, uintptr_t logits, int batch,
                           int in_f, int out_f, uintptr_t s) {
        linear_fwd(ptr<const bf16_raw>(x), ptr<const float>(w), ptr<const float>(b),
                   ptr<float>(logits), batch, in_f, out_f, st(s));
    });
    m.def("linear_bwd", [](uintptr_t x, uintptr_t w, uintptr_t dl, uintptr_t dw, uintptr_t db,
                           uintptr_t dx, int batch, int in_f, int out_f, uintptr_t s) {
        linear_bwd(ptr<const bf16_raw>(x), ptr<const float>(w), ptr<const float>(dl),
                   ptr<float>(dw), ptr<float>(db), ptr<bf16_raw>(dx), batch, in_f, out_f, st(s));
    });
    m.def("softmax_xent", [](uintptr_t logits, uintptr_t target, uintptr_t loss, uintptr_t dl,
                             uintptr_t correct, int batch, int classes, float gscale, uintptr_t s) {
        softmax_xent(ptr<const float>(logits), ptr<const int64_t>(target), ptr<float>(loss),
                     ptr<float>(dl), ptr<int32_t>(correct), batch, classes, gscale, st(s));
    });
    m.def("sgd_momentum", [](uintptr_t p, uintptr_t g, uintptr_t mom, uintptr_t shadow, size_t n,
                             float lr, float mu, float wd, float gscale, bool first, uintptr_t s) {
        sgd_momentum(ptr<float>(p), ptr<const float>(g), ptr<float>(mom), ptr<bf16_raw>(shadow), n,
                     lr, mu, wd, gscale, first, st(s));
    });
    // matrices: (rows, cols, batch, offset, ld, stride, out_offset, out_ld, out_stride, lr) each
    typedef std::tuple<int, int, int, long long, long long, long long, long long, long long, long long,
                       float> NsTuple;
    py::class_<NewtonSchulzPlan>(m, "NewtonSchulzPlan")
        .def(py::init([](const std::vector<NsTuple>& matrices,
                         const std::vector<std::pair<long long, long long>>& segments,
                         const std::vector<float>& coefficients, double eps, bool wide_products) {
            std::vector<NsShape> shapes;
            for (const NsTuple& t : matrices) {
                NsShape s;
                std::tie(s.rows, s.cols, s.batch, s.offset, s.ld, s.stride, s.out_offset, s.out_ld,
                         s.out_stride, s.lr) = t;
                shapes.push_back(s);
            }
            std::vector<NsSegment> segs;
            for (const auto& g : segments) segs.push_back(NsSegment{g.first, g.second});
            return new NewtonSchulzPlan(shapes, segs, coefficients, eps, wide_products);
        }))
        .def_property_readonly("workspace_bytes", &NewtonSchulzPlan::workspace_bytes)
        // (kernel, tile, blocks, threads, tiles made whole, tiles joined from parts) each
        .def_property_readonly("launches", [](const NewtonSchulzPlan& n) {
            std::vector<std::tuple<std::string, std::string, unsigned, unsigned, unsigned, unsigned>> out;
            for (const NsLaunchInfo& l : n.launches())
                out.emplace_back(l.kernel, l.tile, l.blocks, l.threads, l.whole, l.joined);
            return out;
        })
        .def("orthogonalize", [](const NewtonSchulzPlan& n, uintptr_t x, uintptr_t out, int type,
                                 uintptr_t ws, size_t ws_bytes, uintptr_t s) {
            if (type < NS_F32 || type > NS_F16) throw std::invalid_argument("newton_schulz: element type");
            n.orthogonalize(ptr<const void>(x), ptr<void>(out), (NsType)type, ptr<void>(ws), ws_bytes, st(s));
        })
        .def("muon", [](const NewtonSchulzPlan& n, uintptr_t p, uintptr_t g, uintptr_t mom, float lr,
                        float momentum, float weight_decay, bool nesterov, float sgd_lr,
                        float sgd_momentum, float sgd_weight_decay, float grad_scale, uintptr_t ws,
                        size_t ws_bytes, uintptr_t s) {
            MuonArgs a;
            a.lr = lr; a.momentum = momentum; a.weight_decay = weight_decay; a.nesterov = nesterov;
            a.sgd_lr = sgd_lr; a.sgd_momentum = sgd_momentum; a.sgd_weight_decay = sgd_weight_decay;
            a.grad_scale = grad_scale;
            n.muon(ptr<float>(p), ptr<const float>(g), ptr<float>(mom), a, ptr<void>(ws), ws_bytes, st(s));
        });
    m.def("cast_f32_to_bf16", [](uintptr_t x, uintptr_t out, size_t n, uintptr_t s) {
        cast_f32_to_bf16(ptr<const float>(x), ptr<bf16_raw>(out), n, st(s));
    });
    m.def("cast_bf16_to_f32", [](uintptr_t x, uintptr_t out, size_t n, uintptr_t s) {
        cast_bf16_to_f32(ptr<const bf16_raw>(x), ptr<float>(out), n, st(s));
    });
    m.def("augment_normalize", [](uintptr_t img, uintptr_t aug, uintptr_t out, int batch,
                                  std::vector<float> mean, std::vector<float> stdv, uintptr_t s) {
        if (mean.size() != 3 || stdv.size() != 3) throw std::invalid_argument("mean/std need 3");
        augment_normalize(ptr<const uint8_t>(img), ptr<const int32_t>(aug), ptr<bf16_raw>(out),
                          batch, mean.data(), stdv.data(), st(s));
    });
    m.def("nchw_to_nhwc4", [](uintptr_t x, uintptr_t out, int batch, uintptr_t s) {
        nchw_to_nhwc4(ptr<const float>(x), ptr<bf16_raw>(out), batch, st(s));
    });
    m.def("nchw_f32_to_nhwc_bf16", [](uintptr_t x, uintptr_t out, int b, int c, int hw, uintptr_t s) {
        nchw_f32_to_nhwc_bf16(ptr<const float>(x), ptr<bf16_raw>(out), b, c, hw, st(s));
    });
    m.def("nhwc_bf16_to_nchw_f32", [](uintptr_t x, uintptr_t out, int b, int c, int hw, uintptr_t s) {
        nhwc_bf16_to_nchw_f32(ptr<const bf16_raw>(x), ptr<float>(out), b, c, hw, st(s));
    });
    m.def("sum_slabs", [](uintptr_t slabs, int world, size_t n, uintptr_t s) {
        sum_slabs(ptr<float>(slabs), world, n, st(s));
    });
    m.def("copy_batch", [](std::vector<std::tuple<uintptr_t, uintptr_t, size_t>> items, uintptr_t s) {
        CopyJobs jobs;
        for (const auto& it : items) {
            if (jobs.n == CopyJobs::kMax) { copy_batch(jobs, st(s)); jobs.n = 0; }
            jobs.dst[jobs.n] = (void*)std::get<0>(it);
            jobs.src[jobs.n] = (const void*)std::get<1>(it);
            jobs.bytes[jobs.n] = std::get<2>(it);
            ++jobs.n;
        }
        copy_batch(jobs, st(s));
    });
    m.def("fill_uniform_bf16", [](uintptr_t out, size_t n, uint32_t seed, float scale, uintptr_t s) {
        fill_uniform_bf16(ptr<bf16_raw>(out), n, seed, scale, st(s));
    });

    // ------------------------------------------------------ fp32-activation kernels
    m.def("conv3x3_igemm_f32", [](uintptr_t x, uintptr_t w, uintptr_t y, uintptr_t bias,
                                  uintptr_t mask, int batch, int hw, int cin, int cout, int epi,
                                  uintptr_t stream, int tile, int pm, int split) {
        conv3x3_igemm_f32(ptr<const float>(x), ptr<const float>(w), ptr<float>(y),
                          ptr<const float>(bias), ptr<const float>(mask),
                          shape(batch, hw, cin, cout), (ConvEpilogue)epi, st(stream), tile, pm, split);
    }, py::arg("x"), py::arg("w"), py::arg("y"), py::arg("bias"), py::arg("mask"), py::arg("batch"),
       py::arg("hw"), py::arg("cin"), py::arg("cout"), py::arg("epi"), py::arg("stream"),
       py::arg("tile") = 0, py::arg("pm") = -1, py::arg("split") = -1);
    m.def("repack_dgrad_weights_f32", [](uintptr_t wf, uintptr_t wd, int cout, int cin, uintptr_t s) {
        repack_dgrad_weights_f32(ptr<const float>(wf), ptr<float>(wd), cout, cin, st(s));
    });
    m.def("conv3x3_wgrad_f32", [](uintptr_t x, uintptr_t dy, uintptr_t dw, int batch, int hw,
                                  int cin, int cout, uintptr_t slab, uintptr_t stream, int splits,
                                  int pm) {
        conv3x3_wgrad_f32(ptr<const float>(x), ptr<const float>(dy), ptr<float>(dw),
                          shape(batch, hw, cin, cout), ptr<float>(slab), st(stream), splits, pm);
    }, py::arg("x"), py::arg("dy"), py::arg("dw"), py::arg("batch"), py::arg("hw"), py::arg("cin"),
       py::arg("cout"), py::arg("slab"), py::arg("stream"), py::arg("splits") = 0,
       py::arg("pm") = -1);
    m.def("conv3x3_wgrad_f32_splits", [](int batch, int hw, int cin, int cout, int force, int pm) {
        return conv3x3_wgrad_f32_splits(shape(batch, hw, cin, cout), force, pm);
    }, py::arg("batch"), py::arg("hw"), py::arg("cin"), py::arg("cout"), py::arg("force") = 0,
       py::arg("pm") = -1);
    m.def("conv1_fprop_f32", [](uintptr_t x, uintptr_t w, uintptr_t bias, uintptr_t y, int batch,
                                bool relu, uintptr_t s) {
        conv1_fprop_f32(ptr<const float>(x), ptr<const float>(w), ptr<const float>(bias),
                        ptr<float>(y), batch, relu, st(s));
    });
    m.def("conv1_wgrad_f32", [](uintptr_t x, uintptr_t dy, uintptr_t dw, uintptr_t db, int batch,
                                uintptr_t ws, uintptr_t s) {
        conv1_wgrad_f32(ptr<const float>(x), ptr<const float>(dy), ptr<float>(dw), ptr<float>(db),
                        batch, ptr<float>(ws), st(s));
    });
    m.def("conv1_wgrad_f32_workspace_elems", &conv1_wgrad_f32_workspace_elems);
    m.def("relu_mask", [](uintptr_t x, uintptr_t mask, uintptr_t y, size_t n, uintptr_t s) {
        relu_mask(ptr<const bf16_raw>(x), ptr<const bf16_raw>(mask), ptr<bf16_raw>(y), n, st(s));
    });
    m.def("relu_mask_f32", [](uintptr_t x, uintptr_t mask, uintptr_t y, size_t n, uintptr_t s) {
        relu_mask_f32(ptr<const float>(x), ptr<const float>(mask), ptr<float>(y), n, st(s));
    });
    m.def("maxpool2x2_fwd_f32", [](uintptr_t x, uintptr_t y, int batch, int hw, int c, uintptr_t s) {
        maxpool2x2_fwd(ptr<const float>(x), ptr<float>(y), batch, hw, c, st(s));
    });
    m.def("maxpool2x2_bwd_f32", [](uintptr_t x, uintptr_t dy, uintptr_t dx, int batch, int hw, int c,
                                   bool relu_mask, uintptr_t s) {
        maxpool2x2_bwd(ptr<const float>(x), ptr<const float>(dy), ptr<float>(dx), batch, hw, c,
                       relu_mask, st(s));
    });
    m.def("column_sum_f32", [](uintptr_t x, uintptr_t out, int rows, int cols, uintptr_t ws,
                               uintptr_t s) {
        column_sum(ptr<const float>(x), ptr<float>(out), rows, cols, ptr<float>(ws), st(s));
    });
    m.def("bn_relu_fwd_train_f32", [](uintptr_t x, uintptr_t y, uintptr_t gamma, uintptr_t beta,
                                      uintptr_t rm, uintptr_t rv, uintptr_t smean, uintptr_t srstd,
                                      uintptr_t ws, int rows, int c, float momentum, float eps,
                                      uintptr_t s) {
        bn_relu_fwd_train(ptr<const float>(x), ptr<float>(y), ptr<const float>(gamma),
                          ptr<const float>(beta), ptr<float>(rm), ptr<float>(rv), ptr<float>(smean),
                          ptr<float>(srstd), ptr<float>(ws), rows, c, momentum, eps, st(s));
    });
    m.def("bn_relu_fwd_eval_f32", [](uintptr_t x, uintptr_t y, uintptr_t gamma, uintptr_t beta,
                                     uintptr_t rm, uintptr_t rv, int rows, int c, float eps,
                                     uintptr_t s) {
        bn_relu_fwd_eval(ptr<const float>(x), ptr<float>(y), ptr<const float>(gamma),
                         ptr<const float>(beta), ptr<const float>(rm), ptr<const float>(rv), rows,
                         c, eps, st(s));
    });
    m.def("bn_relu_bwd_f32", [](uintptr_t x, uintptr_t dy, uintptr_t dx, uintptr_t gamma,
                                uintptr_t beta, uintptr_t smean, uintptr_t srstd, uintptr_t dgamma,
                                uintptr_t dbeta, uintptr_t ws, int rows, int c, uintptr_t s) {
        bn_relu_bwd(ptr<const float>(x), ptr<float>(dy), ptr<float>(dx), ptr<const float>(gamma),
                    ptr<const float>(beta), ptr<const float>(smean), ptr<const float>(srstd),
                    ptr<float>(dgamma), ptr<float>(dbeta), ptr<float>(ws), rows, c, st(s));
    });
    m.def("bn_relu_pool_fwd_train_f32", [](uintptr_t x, uintptr_t y, uintptr_t gamma, uintptr_t beta,
                                           uintptr_t rm, uintptr_t rv, uintptr_t smean,
                                           uintptr_t srstd, uintptr_t ws, int batch, int hw, int c,
                                           float momentum, float eps, uintptr_t s) {
        bn_relu_pool_fwd_train(ptr<const float>(x), ptr<float>(y), ptr<const float>(gamma),
                               ptr<const float>(beta), ptr<float>(rm), ptr<float>(rv),
                               ptr<float>(smean), ptr<float>(srstd), ptr<float>(ws), batch, hw, c,
                               momentum, eps, st(s));
    });
    m.def("bn_relu_pool_fwd_eval_f32", [](uintptr_t x, uintptr_t y, uintptr_t gamma, uintptr_t beta,
                                          uintptr_t rm, uintptr_t rv, int batch, int hw, int c,
                                          float eps, uintptr_t s) {
        bn_relu_pool_fwd_eval(ptr<const float>(x), ptr<float>(y), ptr<const float>(gamma),
                              ptr<const float>(beta), ptr<const float>(rm), ptr<const float>(rv),
                              batch, hw, c, eps, st(s));
    });
    m.def("bn_relu_pool_bwd_f32", [](uintptr_t x, uintptr_t dy, uintptr_t dx, uintptr_t gamma,
                                     uintptr_t beta, uintptr_t smean, uintptr_t srstd,
                                     uintptr_t dgamma, uintptr_t dbeta, uintptr_t ws, int batch,
                                     int hw, int c, uintptr_t s) {
        bn_relu_pool_bwd(ptr<const float>(x), ptr<float>(dy), ptr<float>(dx), ptr<const float>(gamma),
                         ptr<const float>(beta), ptr<const float>(smean), ptr<const float>(srstd),
                         ptr<float>(dgamma), ptr<float>(dbeta), ptr<float>(ws), batch, hw, c, st(s));
    });
    m.def("linear_fwd_f32", [](uintptr_t x, uintptr_t w, uintptr_t b, uintptr_t logits, int batch,
                               int in_f, int out_f, uintptr_t s) {
        linear_fwd(ptr<const float>(x), ptr<const float>(w), ptr<const float>(b),
                   ptr<float>(logits), batch, in_f, out_f, st(s));
    });
    m.def("fc_train_f32", [](uintptr_t x, uintptr_t w, uintptr_t b, uintptr_t target,
                             uintptr_t logits, uintptr_t loss, uintptr_t correct, uintptr_t dx,
                             uintptr_t dw, uintptr_t db, uintptr_t ws, int batch, int in_f,
                             int out_f, uintptr_t s) {
        fc_train_rows(ptr<const float>(x), ptr<const float>(w), ptr<const float>(b),
                      ptr<const int64_t>(target), ptr<float>(logits), ptr<float>(dx),
                      ptr<float>(ws), batch, in_f, out_f, st(s));
        fc_train_grads(ptr<const float>(x), ptr<const float>(ws), ptr<float>(loss),
                       ptr<int32_t>(correct), ptr<float>(dw), ptr<float>(db), batch, in_f, out_f,
                       st(s));
    });
    m.def("augment_normalize_f32", [](uintptr_t img, uintptr_t aug, uintptr_t out, int batch,
                                      std::vector<float> mean, std::vector<float> stdv,
                                      uintptr_t s) {
        if (mean.size() != 3 || stdv.size() != 3) throw std::invalid_argument("mean/std need 3");
        augment_normalize(ptr<const uint8_t>(img), ptr<const int32_t>(aug), ptr<float>(out), batch,
                          mean.data(), stdv.data(), st(s));
    });
    m.def("nchw_to_nhwc4_f32", [](uintptr_t x, uintptr_t out, int batch, uintptr_t s) {
        nchw_to_nhwc4(ptr<const float>(x), ptr<float>(out), batch, st(s));
    });

    // ------------------------------------------------------------- communication
    bind_comm(m);
    // -------------------------------------------------------------------- engine
    bind_engine(m);
    bind_engine_f32(m);
}
