// torch_ops.cpp -- the eager host path of dibr_rasterization (and of the tutorial loop's other
// library ops: prepare_vertices, mask_iou, texture_mapping; and the sequence operators over packs)
// as compiled autograd nodes.
//
// The reference's native layer is a compiled extension (kaolin/csrc/bindings.cpp); its Python
// front-end (render/mesh/dibr.py:119-209) pays one autograd Function per op.  The ctypes route of
// kaolin/_fused.py costs ~45 us of Python per direction at cfg3 (13 output allocations, ~30
// ctypes arguments, the autograd Function's Python forward and backward) -- as much as the GPU
// work on a slow host.  This file is the same DibrRasterizationCuda node in C++: at::empty for the
// outputs and the compact soft-mask state, the C ABI (include/kaolin_hip.h) called directly, the
// backward run by the autograd engine without re-entering Python.  Results are those of
// kl_dibr_forward / kl_dibr_backward, i.e. bit-identical to the Python path
// (tests/test_gpu_parity.py::test_compiled_node_equals_python_node).
//
// Plumbing only: no torch types cross the C ABI; the stream is the caller's current HIP stream,
// passed in as a handle (torch._C._cuda_getCurrentRawStream) and kept for the backward, which the
// autograd engine runs on the forward's stream.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>

#include <cmath>
#include <map>
#include <mutex>
#include <string>
#include <tuple>

#include "kaolin_hip.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int rc, const char *func) {
  if (rc != 0) throw std::runtime_error(std::string(func) + ": " + kl_last_error() + " (kaolin HIP error " +
                                        std::to_string(rc) + ")");
}

kl_dtype dtype_code(at::ScalarType t) {
  if (t == at::kFloat) return KL_F32;
  if (t == at::kDouble) return KL_F64;
  throw std::runtime_error("kaolin compiled node: f32 / f64 only");
}

// scratch reused across calls on one (device, stream), grown to the largest request: every entry
// point treats its workspace as uninitialised and is done with it when the stream reaches the
// call's end (the Python path's _native.workspace).  A call being captured into a graph gets its
// own buffer from the graph's memory pool instead (graphs replayed concurrently do not share it,
// and a later, larger request cannot free what a graph points at).
at::Tensor workspace(size_t bytes, const at::Device &dev, int64_t stream) {
  if (kl_stream_is_capturing((kl_stream)stream))
    return at::empty({(int64_t)std::max<size_t>(bytes, 16)}, at::TensorOptions().dtype(at::kByte).device(dev));
  static std::mutex mu;
  static std::map<std::pair<int, int64_t>, at::Tensor> cache;
  std::lock_guard<std::mutex> lock(mu);
  at::Tensor &t = cache[{dev.index(), stream}];
  const int64_t need = (int64_t)std::max<size_t>(bytes, 16);
  if (!t.defined() || t.numel() < need) t = at::empty({need}, at::TensorOptions().dtype(at::kByte).device(dev));
  return t;
}

// a buffer that is zero whenever the stream reaches a call that uses it, and that the call leaves
// zero (kl_dibr_backward's soft accumulator): zeroed once when allocated, per (device, stream);
// a captured call gets its own, zeroed by a fill recorded in the graph (_native.zero_kept)
at::Tensor zero_kept(size_t bytes, const at::Device &dev, int64_t stream) {
  const int64_t need = (int64_t)std::max<size_t>(bytes, 16);
  if (kl_stream_is_capturing((kl_stream)stream)) return at::zeros({need}, at::TensorOptions().dtype(at::kByte).device(dev));
  static std::mutex mu;
  static std::map<std::pair<int, int64_t>, at::Tensor> cache;
  std::lock_guard<std::mutex> lock(mu);
  at::Tensor &t = cache[{dev.index(), stream}];
  if (!t.defined() || t.numel() < need) t = at::zeros({need}, at::TensorOptions().dtype(at::kByte).device(dev));
  return t;
}

void *ptr(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// Each node's backward is one opaque HIP call, so its gradients cannot be differentiated again.
// dibr_rasterization (whose reference backward is a CUDA kernel too) raises under create_graph
// (grad mode on inside the backward) rather than hand back gradients that silently drop its
// second-order term.  The nodes whose reference is plain torch (mask_iou, prepare_vertices,
// texture_mapping) instead take the reference chain's own differentiable gradient then
// (the *_chain functions below), as the reference would give.
void no_double_backward(const char *op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op,
              ": backward with create_graph=True is not supported (the backward is one HIP call and is not "
              "differentiable)");
}

// The reference's torch chains (kaolin/_double_backward.py restates them for the Python nodes), in
// ATen ops: the same kernels the Python front-ends' torch fallbacks dispatch to, so the gradients
// taken through them are the reference's.  No Python here: the backward runs on the autograd
// engine's device thread.
// Every op is its own statement, in the order Python evaluates the reference's expressions: the
// autograd engine orders the adds of a tensor's gradients by node creation order, and C++ leaves
// the order of a call's argument expressions unspecified.
at::Tensor mask_iou_chain(const at::Tensor &lhs, const at::Tensor &rhs) {  // metrics/render.py:34-37
  const int64_t B = lhs.size(0);
  const at::Tensor sil_mul = lhs * rhs;
  const at::Tensor sil_add = lhs + rhs;
  const at::Tensor up = at::sum(sil_mul.reshape({B, -1}), 1);
  const at::Tensor diff = sil_add - sil_mul;
  const at::Tensor down = at::sum(diff.reshape({B, -1}), 1);
  const at::Tensor den = down + 1e-10;
  const at::Tensor iou = up / den;
  return at::rsub(at::mean(iou), 1.0);
}

at::Tensor by_faces(const at::Tensor &x, const at::Tensor &faces) {  // index_vertices_by_faces
  const at::Tensor inp = x.unsqueeze(2).expand({-1, -1, faces.size(-1), -1});
  const at::Tensor idx = faces.unsqueeze(0).unsqueeze(-1).expand({x.size(0), -1, -1, x.size(-1)});
  return at::gather(inp, 1, idx);
}

// render/mesh/utils.py:160-175 (rotate_translate_points / pad @ transform, perspective_camera,
// index_vertices_by_faces, face_normals(unit=True))
std::vector<at::Tensor> prepare_chain(const at::Tensor &v, const at::Tensor &faces, const at::Tensor &proj,
                                      const at::Tensor &rot, const at::Tensor &trans, const at::Tensor &xf) {
  at::Tensor vc;
  if (xf.defined()) {
    const at::Tensor padded = at::constant_pad_nd(v, {0, 1}, 1.0);
    vc = at::matmul(padded, xf);
  } else {
    const at::Tensor tv = trans.view({-1, 1, 3});
    const at::Tensor translated = v - tv;
    const at::Tensor rt = rot.permute({0, 2, 1});
    vc = at::matmul(translated, rt);
  }
  const at::Tensor pv = proj.view({-1, 1, 3});
  const at::Tensor pp = vc * pv;
  const at::Tensor pxy = pp.slice(2, 0, 2);
  const at::Tensor pz = pp.slice(2, 2, 3);
  const at::Tensor vi = pxy / pz;
  const at::Tensor fvc = by_faces(vc, faces);
  const at::Tensor fvi = by_faces(vi, faces);
  const at::Tensor c1 = fvc.select(2, 1);
  const at::Tensor c0 = fvc.select(2, 0);
  const at::Tensor e0 = c1 - c0;
  const at::Tensor c2 = fvc.select(2, 2);
  const at::Tensor c0b = fvc.select(2, 0);
  const at::Tensor e1 = c2 - c0b;
  const at::Tensor n = at::cross(e0, e1, 2);
  const at::Tensor len = at::linalg_vector_norm(n, 2, at::IntArrayRef{2}, true);
  const at::Tensor den = len + 1e-10;
  return {fvc, fvi, n / den};
}

at::Tensor texture_chain(const at::Tensor &coords, const at::Tensor &tex, int64_t mode) {  // utils.py:64-75
  const int64_t B = coords.size(0);
  const at::Tensor cl = at::clamp(coords.reshape({B, -1, 1, 2}), 0., 1.);
  const at::Tensor c2 = cl * 2;
  at::Tensor c = c2 - 1;
  const at::Tensor ny = -c.select(3, 1);
  c.select(3, 1).copy_(ny);
  const at::Tensor out = at::grid_sampler(tex, c, mode == 1 ? 0 : 1, /*border*/ 1, false);
  return out.permute({0, 2, 3, 1}).reshape({B, -1, tex.size(1)});
}

// d outputs / d inputs with the graph kept (create_graph): undefined where an input needs none
variable_list chain_grads(const variable_list &outs, const variable_list &gouts, const variable_list &inputs) {
  variable_list live, o, g;
  for (const auto &x : inputs)
    if (x.defined() && x.requires_grad()) live.push_back(x);
  for (size_t k = 0; k < outs.size(); k++)
    if (gouts[k].defined()) {
      o.push_back(outs[k]);
      g.push_back(gouts[k]);
    }
  variable_list res(inputs.size());
  if (live.empty() || o.empty()) return res;
  const variable_list got = torch::autograd::grad(o, live, g, /*retain_graph=*/true, /*create_graph=*/true,
                                                  /*allow_unused=*/true);
  size_t j = 0;
  for (size_t k = 0; k < inputs.size(); k++)
    if (inputs[k].defined() && inputs[k].requires_grad()) res[k] = got[j++];
  return res;
}

struct DibrRasterization : public torch::autograd::Function<DibrRasterization> {
  static variable_list forward(AutogradContext *ctx, int64_t height, int64_t width, at::Tensor fvz, at::Tensor fvi,
                               at::Tensor feat, at::Tensor fnz, double sigmainv, double boxlen, int64_t knum,
                               double multiplier, double eps, int64_t stream) {
    fvz = fvz.contiguous();
    fvi = fvi.contiguous();
    feat = feat.contiguous();
    fnz = fnz.detach().contiguous();
    // one dtype for every float input: the kernels read all of them as fvi's type
    TORCH_CHECK(fvz.scalar_type() == fvi.scalar_type() && feat.scalar_type() == fvi.scalar_type() &&
                    fnz.scalar_type() == fvi.scalar_type(),
                "dibr_rasterization: face_vertices_z, face_vertices_image, face_features and face_normals_z must "
                "share one dtype");
    const int64_t B = fvz.size(0), F = fvz.size(1), D = feat.size(-1);
    const int H = (int)height, W = (int)width, K = (int)knum;
    const auto opt = fvi.options();
    const auto dev = fvi.device();
    const kl_dtype dt = dtype_code(fvi.scalar_type());
    at::Tensor feats = at::empty({B, H, W, D}, opt);
    at::Tensor idx = at::empty({B, H, W}, opt.dtype(at::kLong));
    at::Tensor w = at::empty({B, H, W, 3}, opt);
    at::Tensor mask = at::empty({B, H, W}, opt);
    at::Tensor hits = at::empty({B, H, W}, opt.dtype(at::kByte));
    const int64_t nrec = std::max<int64_t>((int64_t)kl_soft_mask_compact_records((int)B, H, W, K), 1);
    at::Tensor rec_face = at::empty({nrec}, opt.dtype(at::kInt));
    at::Tensor rec_prob = at::empty({nrec}, opt);
    at::Tensor seg_tot =
        at::empty({std::max<int64_t>((int64_t)kl_soft_mask_compact_segments((int)B, H, W), 1)}, opt.dtype(at::kInt));
    // the backward's soft-mask work items (written by the forward)
    at::Tensor scratch = at::empty({(int64_t)kl_dibr_state_bytes((int)B, H, W, (int)F, K)}, opt.dtype(at::kByte));
    at::Tensor ranges = at::empty({B, F, 2}, opt.dtype(at::kInt));
    const size_t nbytes = kl_dibr_workspace_bytes((int)B, H, W, (int)F);
    at::Tensor ws = workspace(nbytes, dev, stream);
    check(kl_dibr_forward(dt, (int)B, H, W, (int)F, (int)D, K, ptr(fvz), ptr(fvi), ptr(feat), ptr(fnz), (float)sigmainv,
                          boxlen * multiplier, (float)multiplier, (float)eps, ptr(feats), idx.data_ptr<int64_t>(),
                          ptr(w), ptr(mask), hits.data_ptr<uint8_t>(), (uint32_t *)rec_face.data_ptr(), ptr(rec_prob),
                          seg_tot.data_ptr<int>(), scratch.data_ptr(),
                          F > 0 ? (uint32_t *)ranges.data_ptr() : nullptr, ws.data_ptr(), nbytes,
                          (kl_stream)stream),
          "dibr_rasterization");
    ctx->mark_non_differentiable({idx});
    ctx->set_materialize_grads(false);
    ctx->saved_data["sigmainv"] = sigmainv;
    ctx->saved_data["multiplier"] = multiplier;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["knum"] = knum;
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["has_ranges"] = F > 0;
    ctx->save_for_backward({idx, w, fvi, feat, fnz, mask, ranges, hits, rec_face, rec_prob, seg_tot, scratch});
    return {feats, mask, idx};
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &idx = saved[0], &w = saved[1], &fvi = saved[2], &feat = saved[3], &fnz = saved[4],
                     &mask = saved[5], &ranges = saved[6], &hits = saved[7], &rec_face = saved[8],
                     &rec_prob = saved[9], &seg_tot = saved[10], &scratch = saved[11];
    no_double_backward("dibr_rasterization");
    at::Tensor gf = grads[0], gm = grads[1];
    variable_list out(12);
    if (!gf.defined() && !gm.defined()) return out;
    if (!gf.defined()) gf = at::zeros({idx.size(0), idx.size(1), idx.size(2), feat.size(-1)}, feat.options());
    gf = gf.contiguous();
    if (gm.defined()) gm = gm.contiguous();
    const int64_t B = fvi.size(0), F = fvi.size(1), D = feat.size(-1);
    const int H = (int)idx.size(1), W = (int)idx.size(2), K = (int)ctx->saved_data["knum"].toInt();
    const int64_t stream = ctx->saved_data["stream"].toInt();
    at::Tensor g_img = at::empty_like(fvi);
    at::Tensor g_feat = at::empty_like(feat);
    const size_t nbytes = kl_dibr_bwd_workspace_bytes((int)B, H, W, (int)F, K);
    at::Tensor ws = workspace(nbytes, fvi.device(), stream);
    at::Tensor acc = gm.defined() ? zero_kept(kl_dibr_soft_acc_bytes((int)B, (int)F), fvi.device(), stream) : at::Tensor();
    check(kl_dibr_backward(dtype_code(fvi.scalar_type()), (int)B, H, W, (int)F, (int)D, K, ptr(gf), ptr(gm),
                           idx.data_ptr<int64_t>(), ptr(w), ptr(fvi), ptr(feat), ptr(fnz), ptr(mask),
                           hits.data_ptr<uint8_t>(), (const uint32_t *)rec_face.data_ptr(), ptr(rec_prob),
                           seg_tot.data_ptr<int>(), (float)ctx->saved_data["sigmainv"].toDouble(),
                           (float)ctx->saved_data["multiplier"].toDouble(), (float)ctx->saved_data["eps"].toDouble(),
                           ptr(g_img), ptr(g_feat), scratch.data_ptr(),
                           ctx->saved_data["has_ranges"].toBool() ? (const uint32_t *)ranges.data_ptr() : nullptr,
                           ptr(acc), ws.data_ptr(), nbytes, (kl_stream)stream),
          "dibr_rasterization backward");
    out[3] = g_img;
    out[4] = g_feat;
    return out;
  }
};

// mask_iou (metrics/render.py MaskIouHip): kl_mask_iou_forward / _backward
struct MaskIou : public torch::autograd::Function<MaskIou> {
  static variable_list forward(AutogradContext *ctx, at::Tensor lhs_in, at::Tensor rhs_in, int64_t stream) {
    const at::Tensor lhs = lhs_in.contiguous(), rhs = rhs_in.contiguous();
    const int64_t B = lhs.size(0), n = lhs.numel() / B;
    const auto opt = lhs.options();
    at::Tensor up = at::empty({B}, opt), down = at::empty({B}, opt), loss = at::empty({}, opt);
    const size_t nbytes = kl_mask_iou_workspace_bytes((int)B, n);
    at::Tensor ws = workspace(nbytes, lhs.device(), stream);
    check(kl_mask_iou_forward(dtype_code(lhs.scalar_type()), (int)B, n, ptr(lhs), ptr(rhs), ptr(up), ptr(down),
                              ptr(loss), ws.data_ptr(), nbytes, (kl_stream)stream),
          "mask_iou");
    ctx->saved_data["stream"] = stream;
    ctx->save_for_backward({lhs_in, rhs_in, up, down});  // the inputs themselves (double backward)
    return {loss};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &up = saved[2], &down = saved[3];
    const bool need_l = ctx->needs_input_grad(0), need_r = ctx->needs_input_grad(1);
    variable_list out(3);
    if (!need_l && !need_r) return out;
    at::Tensor g = grads[0].defined() ? grads[0].contiguous() : at::ones({}, saved[0].options());
    if (at::GradMode::is_enabled()) {  // create_graph: the reference's torch gradient
      const auto r = chain_grads({mask_iou_chain(saved[0], saved[1])}, {g}, {saved[0], saved[1]});
      out[0] = r[0];
      out[1] = r[1];
      return out;
    }
    const at::Tensor lhs = saved[0].contiguous(), rhs = saved[1].contiguous();
    at::Tensor gl = need_l ? at::empty_like(lhs) : at::Tensor(), gr = need_r ? at::empty_like(rhs) : at::Tensor();
    const int64_t B = lhs.size(0);
    check(kl_mask_iou_backward(dtype_code(lhs.scalar_type()), (int)B, lhs.numel() / B, ptr(g), ptr(lhs), ptr(rhs),
                               ptr(up), ptr(down), ptr(gl), ptr(gr), (kl_stream)ctx->saved_data["stream"].toInt()),
          "mask_iou backward");
    out[0] = gl;
    out[1] = gr;
    return out;
  }
};

at::Tensor mask_iou(at::Tensor lhs, at::Tensor rhs, int64_t stream) { return MaskIou::apply(lhs, rhs, stream)[0]; }

// prepare_vertices (render/mesh/utils.py PrepareVerticesHip): kl_prepare_vertices_forward / _backward.
// cam_a, cam_b = rot, trans; or xf (camera_transform) twice (has_xf; the second slot gets no
// gradient) -- autograd's apply takes no undefined tensors.  batches (B, Bv, Bc, Bp) as the Python
// front-end computes them.
struct PrepareVertices : public torch::autograd::Function<PrepareVertices> {
  static variable_list forward(AutogradContext *ctx, at::Tensor vertices, at::Tensor faces, at::Tensor proj,
                               at::Tensor cam_a, at::Tensor cam_b, bool has_xf, std::vector<int64_t> batches,
                               int64_t stream) {
    const int64_t B = batches[0], Bv = batches[1], Bc = batches[2], Bp = batches[3];
    at::Tensor verts = vertices.contiguous(), fc = faces.contiguous(), pj = proj.contiguous();
    at::Tensor r = has_xf ? at::Tensor() : cam_a.contiguous(), t = has_xf ? at::Tensor() : cam_b.contiguous();
    at::Tensor x = has_xf ? cam_a.contiguous() : at::Tensor();
    const int64_t V = verts.size(1), F = fc.size(0);
    const auto opt = verts.options();
    at::Tensor fvc = at::empty({B, F, 3, 3}, opt), fvi = at::empty({B, F, 3, 2}, opt), fn = at::empty({B, F, 3}, opt);
    check(kl_prepare_vertices_forward(dtype_code(verts.scalar_type()), (int)B, (int)Bv, (int)Bc, (int)Bp, V, F,
                                      ptr(verts), fc.data_ptr<int64_t>(), ptr(r), ptr(t), ptr(x), ptr(pj), ptr(fvc),
                                      ptr(fvi), ptr(fn), (kl_stream)stream),
          "prepare_vertices");
    ctx->saved_data["batches"] = batches;
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["proj_shape"] = proj.sizes().vec();
    ctx->saved_data["trans_shape"] = has_xf ? std::vector<int64_t>{} : cam_b.sizes().vec();
    ctx->saved_data["has_xf"] = has_xf;
    ctx->set_materialize_grads(false);
    // the inputs themselves (a double backward differentiates the reference's chain of them)
    ctx->save_for_backward({vertices, faces, proj, has_xf ? at::Tensor() : cam_a, has_xf ? at::Tensor() : cam_b,
                            has_xf ? cam_a : at::Tensor()});
    return {fvc, fvi, fn};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    variable_list out(8);
    if (!grads[0].defined() && !grads[1].defined() && !grads[2].defined()) return out;
    const bool has_xf = ctx->saved_data["has_xf"].toBool();
    if (at::GradMode::is_enabled()) {  // create_graph: the reference's torch gradient
      const auto g = chain_grads(prepare_chain(saved[0], saved[1], saved[2], saved[3], saved[4], saved[5]),
                                 {grads[0], grads[1], grads[2]}, {saved[0], saved[2], saved[3], saved[4], saved[5]});
      out[0] = g[0];
      out[2] = g[1];
      out[3] = has_xf ? g[4] : g[2];
      if (!has_xf) out[4] = g[3];
      return out;
    }
    const at::Tensor verts = saved[0].contiguous(), fc = saved[1].contiguous(), pj = saved[2].contiguous();
    const at::Tensor r = saved[3].defined() ? saved[3].contiguous() : at::Tensor();
    const at::Tensor t = saved[4].defined() ? saved[4].contiguous() : at::Tensor();
    const at::Tensor x = saved[5].defined() ? saved[5].contiguous() : at::Tensor();
    const auto b = ctx->saved_data["batches"].toIntVector();
    const int64_t B = b[0], Bv = b[1], Bc = b[2], Bp = b[3];
    const bool need_v = ctx->needs_input_grad(0), need_p = ctx->needs_input_grad(2),
               need_r = !has_xf && ctx->needs_input_grad(3), need_t = !has_xf && ctx->needs_input_grad(4),
               need_x = has_xf && ctx->needs_input_grad(3);
    const auto opt = verts.options();
    at::Tensor g_v = need_v ? at::empty_like(verts) : at::Tensor();
    at::Tensor g_cam = (need_r || need_t || need_x) ? at::empty({Bc, 12}, opt) : at::Tensor();
    at::Tensor g_proj = need_p ? at::empty({Bp, 3}, opt) : at::Tensor();
    const int64_t V = verts.size(1), F = fc.size(0);
    const int64_t stream = ctx->saved_data["stream"].toInt();
    const size_t nbytes = kl_prepare_vertices_bwd_workspace_bytes((int)B, V);
    at::Tensor ws = workspace(nbytes, verts.device(), stream);
    at::Tensor g0 = grads[0].defined() ? grads[0].contiguous() : at::Tensor();
    at::Tensor g1 = grads[1].defined() ? grads[1].contiguous() : at::Tensor();
    at::Tensor g2 = grads[2].defined() ? grads[2].contiguous() : at::Tensor();
    check(kl_prepare_vertices_backward(dtype_code(verts.scalar_type()), (int)B, (int)Bv, (int)Bc, (int)Bp, V, F,
                                       ptr(verts), fc.data_ptr<int64_t>(), ptr(r), ptr(t), ptr(x), ptr(pj), ptr(g0),
                                       ptr(g1), ptr(g2), ptr(g_v), ptr(g_cam), ptr(g_proj), ws.data_ptr(), nbytes,
                                       (kl_stream)stream),
          "prepare_vertices backward");
    out[0] = g_v;
    if (need_p) out[2] = g_proj.reshape(ctx->saved_data["proj_shape"].toIntVector());
    if (need_r) out[3] = g_cam.narrow(1, 0, 9).reshape({Bc, 3, 3});
    if (need_t) out[4] = g_cam.narrow(1, 9, 3).reshape(ctx->saved_data["trans_shape"].toIntVector());
    if (need_x) out[3] = g_cam.reshape({Bc, 4, 3});
    return out;
  }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor> prepare_vertices(at::Tensor vertices, at::Tensor faces, at::Tensor proj,
                                                                c10::optional<at::Tensor> rot,
                                                                c10::optional<at::Tensor> trans,
                                                                c10::optional<at::Tensor> xf,
                                                                std::vector<int64_t> batches, int64_t stream) {
  const bool has_xf = xf.has_value() && xf->defined();
  TORCH_CHECK(has_xf || (rot.has_value() && trans.has_value()), "prepare_vertices: camera_rot and camera_trans, or "
              "camera_transform");
  auto r = has_xf ? PrepareVertices::apply(vertices, faces, proj, *xf, *xf, true, batches, stream)
                  : PrepareVertices::apply(vertices, faces, proj, *rot, *trans, false, batches, stream);
  return {r[0], r[1], r[2]};
}

// texture_mapping (render/mesh/utils.py TextureMappingHip): kl_texture_mapping_forward / _backward
struct TextureMapping : public torch::autograd::Function<TextureMapping> {
  static variable_list forward(AutogradContext *ctx, at::Tensor coords, at::Tensor tex, int64_t mode, int64_t stream) {
    at::Tensor c = coords.contiguous(), t = tex.contiguous();
    const int64_t B = t.size(0), C = t.size(1), TH = t.size(2), TW = t.size(3);
    const int64_t n = B ? c.numel() / (2 * B) : 0;
    at::Tensor out = at::empty({B, n, C}, t.options());
    check(kl_texture_mapping_forward(dtype_code(t.scalar_type()), (int)mode, (int)B, n, (int)C, (int)TH, (int)TW,
                                     ptr(c), ptr(t), ptr(out), (kl_stream)stream),
          "texture_mapping");
    ctx->saved_data["mode"] = mode;
    ctx->saved_data["n"] = n;
    ctx->saved_data["stream"] = stream;
    ctx->save_for_backward({coords, tex});  // the inputs themselves (double backward)
    return {out};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool need_c = ctx->needs_input_grad(0), need_t = ctx->needs_input_grad(1);
    variable_list out(4);
    if ((!need_c && !need_t) || !grads[0].defined()) return out;
    if (at::GradMode::is_enabled()) {  // create_graph: the reference's torch gradient
      const at::Tensor o = texture_chain(saved[0], saved[1], ctx->saved_data["mode"].toInt());
      const auto g = chain_grads({o}, {grads[0].reshape(o.sizes())}, {saved[0], saved[1]});
      out[0] = g[0];
      out[1] = g[1];
      return out;
    }
    const at::Tensor c = saved[0].contiguous(), t = saved[1].contiguous();
    const int64_t B = t.size(0), C = t.size(1), TH = t.size(2), TW = t.size(3);
    const int64_t stream = ctx->saved_data["stream"].toInt();
    at::Tensor gc = need_c ? at::empty_like(c) : at::Tensor(), gt = need_t ? at::empty_like(t) : at::Tensor();
    const size_t nbytes = need_t ? kl_texture_mapping_bwd_workspace_bytes((int)B, (int)C, (int)TH, (int)TW) : 0;
    at::Tensor ws = need_t ? workspace(nbytes, t.device(), stream) : at::Tensor();
    check(kl_texture_mapping_backward(dtype_code(t.scalar_type()), (int)ctx->saved_data["mode"].toInt(), (int)B,
                                      ctx->saved_data["n"].toInt(), (int)C, (int)TH, (int)TW,
                                      ptr(grads[0].contiguous()), ptr(c), ptr(t), ptr(gc), ptr(gt), ptr(ws), nbytes,
                                      (kl_stream)stream),
          "texture_mapping backward");
    out[0] = gc;
    out[1] = gt;
    return out;
  }
};

at::Tensor texture_mapping(at::Tensor coords, at::Tensor tex, int64_t mode, int64_t stream) {
  return TextureMapping::apply(coords, tex, mode, stream)[0];
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> dibr_rasterization(int64_t height, int64_t width, at::Tensor fvz,
                                                                   at::Tensor fvi, at::Tensor feat, at::Tensor fnz,
                                                                   double sigmainv, double boxlen, int64_t knum,
                                                                   double multiplier, double eps, int64_t stream) {
  auto r = DibrRasterization::apply(height, width, fvz, fvi, feat, fnz, sigmainv, boxlen, knum, multiplier, eps,
                                    stream);
  return {r[0], r[1], r[2]};
}

// ---- The sequence operators over packs (kaolin/render/spc/sequence.py, which holds the same nodes in
// Python).  Each function takes the plain case -- types, sizes and strides that the kernels read as they
// are -- and returns nothing for any other call, which the Python route then copies or refuses with its
// message.

kl_dtype seq_code(at::ScalarType t) {
  return t == at::kFloat ? KL_F32 : t == at::kHalf ? KL_F16 : t == at::kBFloat16 ? KL_BF16 : KL_F64;
}

// Scratch of one call alone, from the allocator's pool of the call's stream.  Kernels of a call hand each other numbers
// through it (counts that bound loops among them), and another host thread may launch on the same stream between
// them: a backward runs on the engine's thread.
at::Tensor scratch(size_t bytes, const at::Device &dev) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 16)}, at::TensorOptions().dtype(at::kByte).device(dev));
}

bool seq_float(const at::Tensor &t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16;
}

constexpr int64_t kMaxRows = ((int64_t)1 << 31) - 256;

bool plain_mask(const at::Tensor &b, int64_t rows, const at::Device &dev) {
  return b.dim() == 1 && b.size(0) == rows && rows < kMaxRows && b.device() == dev && b.is_contiguous() &&
         (b.scalar_type() == at::kBool || b.scalar_type() == at::kByte);
}

// (rows, heads, dim) with whole 16-byte pieces in every row of a head
bool plain_heads(const at::Tensor &t) {
  const int64_t e = 16 / t.element_size();
  return t.dim() == 3 && (t.numel() == 0 || (t.stride(2) == 1 && t.stride(0) % e == 0 && t.stride(1) % e == 0 &&
                                             t.stride(0) < (int64_t)1 << 25 && (uintptr_t)t.data_ptr() % 16 == 0));
}

bool any_grad(std::initializer_list<const at::Tensor *> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor *t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// a forward-mode derivative: the Python nodes refuse it, the bare kernels would drop it
bool any_tangent(std::initializer_list<const at::Tensor *> ts) {
  for (const at::Tensor *t : ts)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined()) return true;
  return false;
}

at::Tensor contiguous16(const at::Tensor &t) {
  const at::Tensor c = t.contiguous();
  return c.numel() && (uintptr_t)c.data_ptr() % 16 ? c.clone() : c;
}

// The pack arrays of a mask (kl_pack_layout): ids (n) and starts (n + 1) in one tensor
struct Layout {
  at::Tensor held;
  int32_t *ids() const { return held.data_ptr<int32_t>(); }
  int32_t *starts() const { return held.data_ptr<int32_t>() + (held.numel() - 1) / 2; }
};

Layout make_layout(const at::Tensor &boundaries, int64_t stream) {
  const int64_t n = boundaries.size(0);
  Layout l{at::empty({2 * n + 1}, boundaries.options().dtype(at::kInt))};
  const size_t bytes = kl_pack_layout_workspace_bytes(n);
  at::Tensor ws = scratch(bytes, boundaries.device());
  check(kl_pack_layout(n, (const uint8_t *)boundaries.data_ptr(), l.ids(), l.starts(), ws.data_ptr(), bytes,
                       (kl_stream)stream),
        "pack_layout");
  return l;
}

// of two masks at once
std::pair<Layout, Layout> make_layouts(const at::Tensor &one, const at::Tensor &two, int64_t stream) {
  const int64_t n = one.size(0), m = two.size(0);
  const auto ints = one.options().dtype(at::kInt);
  const Layout a{at::empty({2 * n + 1}, ints)}, b{at::empty({2 * m + 1}, ints)};
  const size_t bytes = kl_pack_layout_workspace_bytes(n) + kl_pack_layout_workspace_bytes(m);
  at::Tensor ws = scratch(bytes, one.device());
  check(kl_pack_layout_pair(n, (const uint8_t *)one.data_ptr(), a.ids(), a.starts(), m, (const uint8_t *)two.data_ptr(),
                            b.ids(), b.starts(), ws.data_ptr(), bytes, (kl_stream)stream),
        "pack_layout_pair");
  return {a, b};
}

struct HeadStrides {
  int64_t v[6];
  HeadStrides(const at::Tensor &q, const at::Tensor &k, const at::Tensor &w)
      : v{q.stride(0), q.stride(1), k.stride(0), k.stride(1), w.stride(0), w.stride(1)} {}
};

std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_forward(const at::Tensor &q, const at::Tensor &k,
                                                                 const at::Tensor &v, const Layout &lq,
                                                                 const Layout &lk, double scale, bool causal,
                                                                 bool for_backward, int64_t stream) {
  const kl_dtype code = seq_code(q.scalar_type());
  at::Tensor out = at::empty(q.sizes(), q.options()), lse, low;
  if (for_backward) {
    lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
    if (code != KL_F32) low = at::empty(q.sizes(), q.options());
  }
  const int heads = (int)q.size(1), kv = (int)k.size(1), dim = (int)q.size(2);
  const size_t bytes = kl_pack_attention_workspace_bytes(code, q.size(0), k.size(0), heads, kv, dim);
  at::Tensor ws = scratch(bytes, q.device());
  const HeadStrides st(q, k, v);
  check(kl_pack_attention_forward(code, q.size(0), k.size(0), heads, kv, dim, ptr(q), ptr(k), ptr(v), st.v, lq.ids(),
                                  lq.starts(), lk.ids(), lk.starts(), (float)scale, causal, ptr(out), ptr(low),
                                  (float *)ptr(lse), ptr(ws), bytes, (kl_stream)stream),
        "pack_attention");
  return {out, lse, low};
}

struct PackAttention : public torch::autograd::Function<PackAttention> {
  static variable_list forward(AutogradContext *ctx, at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor lq,
                               at::Tensor lk, double scale, bool causal, int64_t stream) {
    auto r = attention_forward(q, k, v, Layout{lq}, Layout{lk}, scale, causal, true, stream);
    ctx->save_for_backward({q, k, v, std::get<0>(r), std::get<1>(r), std::get<2>(r), lq, lk});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["stream"] = stream;
    return {std::get<0>(r)};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    no_double_backward("pack_attention");
    variable_list outs(8);
    if (!grads[0].defined()) return outs;
    const auto s = ctx->get_saved_variables();
    const at::Tensor &q = s[0], &k = s[1], &v = s[2];
    const c10::DeviceGuard guard(q.device());
    const bool need_q = ctx->needs_input_grad(0), need_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    const int64_t stream = ctx->saved_data["stream"].toInt();
    const at::Tensor g = contiguous16(grads[0]);
    at::Tensor dq = need_q ? at::empty(q.sizes(), q.options()) : at::Tensor();
    at::Tensor dk = need_kv ? at::empty(k.sizes(), k.options()) : at::Tensor();
    at::Tensor dv = need_kv ? at::empty(v.sizes(), v.options()) : at::Tensor();
    const kl_dtype code = seq_code(q.scalar_type());
    const int heads = (int)q.size(1), kv = (int)k.size(1), dim = (int)q.size(2);
    const size_t bytes = kl_pack_attention_bwd_workspace_bytes(code, q.size(0), k.size(0), heads, kv, dim);
    at::Tensor ws = scratch(bytes, q.device());
    const HeadStrides st(q, k, v);
    const Layout lq{s[6]}, lk{s[7]};
    check(kl_pack_attention_backward(code, q.size(0), k.size(0), heads, kv, dim, ptr(g), ptr(q), ptr(k), ptr(v), st.v,
                                     lq.ids(), lq.starts(), lk.ids(), lk.starts(), ptr(s[3]), ptr(s[5]),
                                     (const float *)ptr(s[4]), (float)ctx->saved_data["scale"].toDouble(),
                                     ctx->saved_data["causal"].toBool(), ptr(dq), ptr(dk), ptr(dv), ptr(ws), bytes,
                                     (kl_stream)stream),
          "pack_attention backward");
    outs[0] = dq;
    if (ctx->needs_input_grad(1)) outs[1] = dk;
    if (ctx->needs_input_grad(2)) outs[2] = dv;
    return outs;
  }
};

c10::optional<at::Tensor> pack_attention(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor boundaries,
                                         c10::optional<at::Tensor> q_boundaries, bool causal, double scale,
                                         int64_t stream) {
  const at::Device dev = q.device();
  const at::Tensor &qb = q_boundaries ? *q_boundaries : boundaries;
  if (!q.is_cuda() || k.device() != dev || v.device() != dev || !seq_float(q) || k.scalar_type() != q.scalar_type() ||
      v.scalar_type() != q.scalar_type() || !plain_heads(q) || !plain_heads(k) || !plain_heads(v) ||
      k.sizes() != v.sizes() || k.size(2) != q.size(2) || q.size(2) % 8 || q.size(2) < 8 || q.size(2) > 128 ||
      k.size(1) == 0 || q.size(1) == 0 || q.size(1) % k.size(1) || q.size(1) > 4096 || !(scale > 0) ||
      !std::isfinite(scale) || !plain_mask(boundaries, k.size(0), dev) || !plain_mask(qb, q.size(0), dev) ||
      any_tangent({&q, &k, &v}))
    return c10::nullopt;
  const c10::DeviceGuard guard(dev);
  Layout lk, lq;
  if (q_boundaries) {
    std::tie(lk, lq) = make_layouts(boundaries, qb, stream);
  } else {
    lk = lq = make_layout(boundaries, stream);
  }
  if (any_grad({&q, &k, &v})) return PackAttention::apply(q, k, v, lq.held, lk.held, scale, causal, stream)[0];
  return std::get<0>(attention_forward(q, k, v, lq, lk, scale, causal, false, stream));
}

// norm_rotary's arguments past q and k
struct NormArgs {
  at::Tensor wq, wk, freqs, held, positions;  // held: a Layout, where positions is not given
  double eps;
  bool interleaved;
  int64_t stream;
  int kind() const {
    if (!positions.defined()) return 0;
    return positions.scalar_type() == at::kInt ? 1 : positions.scalar_type() == at::kLong ? 2 : 3;
  }
  int weight_f32() const { return ((wq.defined() ? wq : wk).defined() &&
                                   (wq.defined() ? wq : wk).scalar_type() == at::kFloat); }
  const int32_t *ids() const { return held.defined() ? Layout{held}.ids() : nullptr; }
  const int32_t *starts() const { return held.defined() ? Layout{held}.starts() : nullptr; }
};

std::pair<at::Tensor, at::Tensor> norm_forward(const at::Tensor &q, const at::Tensor &k, const NormArgs &a) {
  at::Tensor yq = at::empty(q.sizes(), q.options()), yk = at::empty(k.sizes(), k.options());
  const HeadStrides st(q, k, k);
  check(kl_norm_rotary_forward(seq_code(q.scalar_type()), q.size(0), (int)q.size(1), (int)k.size(1), (int)q.size(2),
                               2 * (int)a.freqs.size(0), a.interleaved, ptr(q), ptr(k), st.v, ptr(a.wq), ptr(a.wk),
                               a.weight_f32(), a.freqs.data_ptr<double>(), a.kind(), ptr(a.positions), a.ids(),
                               a.starts(), (float)a.eps, ptr(yq), ptr(yk), (kl_stream)a.stream),
        "norm_rotary");
  return {yq, yk};
}

struct NormRotary : public torch::autograd::Function<NormRotary> {
  using Maybe = c10::optional<at::Tensor>;
  static variable_list forward(AutogradContext *ctx, at::Tensor q, at::Tensor k, Maybe wq_, Maybe wk_, at::Tensor freqs,
                               Maybe held_, Maybe positions_, double eps, bool interleaved, int64_t stream) {
    const at::Tensor wq = wq_.value_or(at::Tensor()), wk = wk_.value_or(at::Tensor()),
                     held = held_.value_or(at::Tensor()), positions = positions_.value_or(at::Tensor());
    auto r = norm_forward(q, k, {wq, wk, freqs, held, positions, eps, interleaved, stream});
    ctx->save_for_backward({q, k, wq, wk, freqs, held, positions});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["stream"] = stream;
    return {r.first, r.second};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    no_double_backward("norm_rotary");
    variable_list outs(10);
    if (!grads[0].defined() && !grads[1].defined()) return outs;
    const auto s = ctx->get_saved_variables();
    const at::Tensor &q = s[0], &k = s[1];
    const c10::DeviceGuard guard(q.device());
    const NormArgs a{s[2], s[3], s[4], s[5], s[6], ctx->saved_data["eps"].toDouble(),
                     ctx->saved_data["interleaved"].toBool(), ctx->saved_data["stream"].toInt()};
    const at::Tensor gq = grads[0].defined() ? contiguous16(grads[0]) : at::zeros(q.sizes(), q.options());
    const at::Tensor gk = grads[1].defined() ? contiguous16(grads[1]) : at::zeros(k.sizes(), k.options());
    at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
    // the inputs that need a gradient are counted without those that are absent
    at::Tensor dwq = a.wq.defined() && ctx->needs_input_grad(2) ? at::empty_like(a.wq) : at::Tensor();
    at::Tensor dwk = a.wk.defined() && ctx->needs_input_grad(a.wq.defined() ? 3 : 2) ? at::empty_like(a.wk)
                                                                                     : at::Tensor();
    const size_t bytes = kl_norm_rotary_bwd_workspace_bytes((int)q.size(2));
    at::Tensor ws = scratch(bytes, q.device());
    const HeadStrides st(q, k, k);
    check(kl_norm_rotary_backward(seq_code(q.scalar_type()), q.size(0), (int)q.size(1), (int)k.size(1), (int)q.size(2),
                                  2 * (int)a.freqs.size(0), a.interleaved, ptr(gq), ptr(gk), ptr(q), ptr(k), st.v,
                                  ptr(a.wq), ptr(a.wk), a.weight_f32(), a.freqs.data_ptr<double>(), a.kind(),
                                  ptr(a.positions), a.ids(), a.starts(), (float)a.eps, ptr(dq), ptr(dk), ptr(dwq),
                                  ptr(dwk), ptr(ws), bytes, (kl_stream)a.stream),
          "norm_rotary backward");
    if (ctx->needs_input_grad(0)) outs[0] = dq;
    if (ctx->needs_input_grad(1)) outs[1] = dk;
    outs[2] = dwq;
    outs[3] = dwk;
    return outs;
  }
};

c10::optional<std::tuple<at::Tensor, at::Tensor>> norm_rotary(at::Tensor q, at::Tensor k, c10::optional<at::Tensor> wq_,
                                                              c10::optional<at::Tensor> wk_, at::Tensor freqs,
                                                              c10::optional<at::Tensor> boundaries,
                                                              c10::optional<at::Tensor> positions_, double eps,
                                                              bool interleaved, int64_t stream) {
  const at::Device dev = q.device();
  const at::Tensor wq = wq_.value_or(at::Tensor()), wk = wk_.value_or(at::Tensor()),
                   positions = positions_.value_or(at::Tensor());
  auto plain_weight = [&](const at::Tensor &w) {
    return !w.defined() || (w.device() == dev && w.dim() == 1 && w.size(0) == q.size(2) && w.is_contiguous() &&
                            (w.scalar_type() == q.scalar_type() || w.scalar_type() == at::kFloat));
  };
  if (!q.is_cuda() || k.device() != dev || !seq_float(q) || k.scalar_type() != q.scalar_type() || !plain_heads(q) ||
      !plain_heads(k) || k.size(0) != q.size(0) || k.size(2) != q.size(2) || q.size(2) % 8 || q.size(2) < 8 ||
      q.size(2) > 256 || q.size(1) + k.size(1) > 1 << 16 || q.size(0) >= kMaxRows || !plain_weight(wq) ||
      !plain_weight(wk) || (wq.defined() && wk.defined() && wq.scalar_type() != wk.scalar_type()) ||
      freqs.device() != dev || freqs.scalar_type() != at::kDouble || freqs.dim() != 1 || !freqs.is_contiguous() ||
      freqs.requires_grad() || 2 * freqs.size(0) > q.size(2) || !(eps >= 0) || !std::isfinite(eps) ||
      boundaries.has_value() == positions.defined() || any_tangent({&q, &k, &wq, &wk, &freqs, &positions}))
    return c10::nullopt;
  if (positions.defined()) {
    const auto t = positions.scalar_type();
    if (positions.device() != dev || positions.dim() != 1 || positions.size(0) != q.size(0) ||
        !positions.is_contiguous() || positions.requires_grad() || (t != at::kInt && t != at::kLong && t != at::kFloat))
      return c10::nullopt;
  } else if (!plain_mask(*boundaries, q.size(0), dev)) {
    return c10::nullopt;
  }
  const c10::DeviceGuard guard(dev);
  c10::optional<at::Tensor> held_;
  if (!positions.defined()) held_ = make_layout(*boundaries, stream).held;
  if (any_grad({&q, &k, &wq, &wk})) {
    auto r = NormRotary::apply(q, k, wq_, wk_, freqs, held_, positions_, eps, interleaved, stream);
    return std::make_tuple(r[0], r[1]);
  }
  const at::Tensor held = held_.value_or(at::Tensor());
  auto r = norm_forward(q, k, {wq, wk, freqs, held, positions, eps, interleaved, stream});
  return std::make_tuple(r.first, r.second);
}

at::Tensor recurrence_forward(const at::Tensor &gates, const at::Tensor &feats, const at::Tensor &initial,
                              const Layout &l, bool reverse, int64_t stream) {
  const kl_dtype code = seq_code(gates.scalar_type());
  const int64_t n = gates.size(0), dim = gates.size(1);
  at::Tensor out = at::empty(gates.sizes(), gates.options());
  const size_t bytes = kl_linear_recurrence_workspace_bytes(code, n, dim);
  at::Tensor ws = scratch(bytes, gates.device());
  check(kl_linear_recurrence_forward(code, n, dim, ptr(gates), ptr(feats), ptr(initial),
                                     initial.defined() ? initial.size(0) : 0, l.ids(), l.starts(), reverse, ptr(out),
                                     ptr(ws), bytes, (kl_stream)stream),
        "linear_recurrence");
  return out;
}

struct LinearRecurrence : public torch::autograd::Function<LinearRecurrence> {
  static variable_list forward(AutogradContext *ctx, at::Tensor gates, at::Tensor feats,
                               c10::optional<at::Tensor> initial_, at::Tensor held, bool reverse, int64_t stream) {
    const at::Tensor initial = initial_.value_or(at::Tensor());
    at::Tensor out = recurrence_forward(gates, feats, initial, Layout{held}, reverse, stream);
    ctx->save_for_backward({gates, out, initial, held});
    ctx->saved_data["reverse"] = reverse;
    ctx->saved_data["stream"] = stream;
    return {out};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    no_double_backward("linear_recurrence");
    variable_list outs(6);
    if (!grads[0].defined()) return outs;
    const auto s = ctx->get_saved_variables();
    const at::Tensor &gates = s[0], &initial = s[2];
    const c10::DeviceGuard guard(gates.device());
    const Layout l{s[3]};
    const int64_t stream = ctx->saved_data["stream"].toInt(), n = gates.size(0), dim = gates.size(1);
    const at::Tensor g = grads[0].contiguous();
    at::Tensor da = at::empty(gates.sizes(), gates.options()), db = at::empty(gates.sizes(), gates.options());
    at::Tensor di = initial.defined() ? at::empty(initial.sizes(), initial.options()) : at::Tensor();
    const kl_dtype code = seq_code(gates.scalar_type());
    const size_t bytes = kl_linear_recurrence_workspace_bytes(code, n, dim);
    at::Tensor ws = scratch(bytes, gates.device());
    check(kl_linear_recurrence_backward(code, n, dim, ptr(g), ptr(gates), ptr(s[1]), ptr(initial),
                                        initial.defined() ? initial.size(0) : 0, l.ids(), l.starts(),
                                        ctx->saved_data["reverse"].toBool(), ptr(da), ptr(db), ptr(di), ptr(ws), bytes,
                                        (kl_stream)stream),
          "linear_recurrence backward");
    if (ctx->needs_input_grad(0)) outs[0] = da;
    if (ctx->needs_input_grad(1)) outs[1] = db;
    if (initial.defined() && ctx->needs_input_grad(2)) outs[2] = di;
    return outs;
  }
};

c10::optional<at::Tensor> linear_recurrence(at::Tensor gates, at::Tensor feats, at::Tensor boundaries,
                                            c10::optional<at::Tensor> initial_, bool reverse, int64_t stream) {
  const at::Device dev = gates.device();
  const at::Tensor initial = initial_.value_or(at::Tensor());
  auto plain = [&](const at::Tensor &t) {
    return t.device() == dev && t.scalar_type() == gates.scalar_type() && t.dim() == 2 && t.is_contiguous();
  };
  if (!gates.is_cuda() || (!seq_float(gates) && gates.scalar_type() != at::kDouble) || !plain(gates) || !plain(feats) ||
      gates.sizes() != feats.sizes() || gates.size(1) >= 1 << 24 || !plain_mask(boundaries, gates.size(0), dev) ||
      (initial.defined() && (!plain(initial) || initial.size(1) != gates.size(1) ||
                             initial.size(0) >= (int64_t)1 << 31)) ||
      any_tangent({&gates, &feats, &initial}))
    return c10::nullopt;
  const c10::DeviceGuard guard(dev);
  const Layout l = make_layout(boundaries, stream);
  if (any_grad({&gates, &feats, &initial}))
    return LinearRecurrence::apply(gates, feats, initial_, l.held, reverse, stream)[0];
  return recurrence_forward(gates, feats, initial, l, reverse, stream);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "kaolin-mi355x compiled autograd nodes over the C ABI (include/kaolin_hip.h)";
  m.def("abi_version", []() { return kl_abi_version(); });
  m.def("dibr_rasterization", &dibr_rasterization,
        "dibr_rasterization's fused node: (features, soft_mask, face_idx); see kaolin/render/mesh/dibr.py");
  m.def("mask_iou", &mask_iou, "mask_iou's fused node; see kaolin/metrics/render.py");
  m.def("prepare_vertices", &prepare_vertices, "prepare_vertices' node; see kaolin/render/mesh/utils.py");
  m.def("texture_mapping", &texture_mapping, "texture_mapping's node; see kaolin/render/mesh/utils.py");
  m.def("pack_attention", &pack_attention, "pack_attention's node, or None; see kaolin/render/spc/sequence.py");
  m.def("norm_rotary", &norm_rotary, "norm_rotary's node, or None; see kaolin/render/spc/sequence.py");
  m.def("linear_recurrence", &linear_recurrence, "linear_recurrence's node, or None; see kaolin/render/spc/sequence.py");
  // the double-backward reference chains, exposed for tests (tests/test_cpu_paths.py)
  m.def("_mask_iou_chain", &mask_iou_chain);
  m.def("_prepare_chain", [](at::Tensor v, at::Tensor faces, at::Tensor proj, c10::optional<at::Tensor> rot,
                             c10::optional<at::Tensor> trans, c10::optional<at::Tensor> xf) {
    return prepare_chain(v, faces, proj, rot.value_or(at::Tensor()), trans.value_or(at::Tensor()),
                         xf.value_or(at::Tensor()));
  });
  m.def("_texture_chain", &texture_chain);
}
