// torch binding `volume_integration._C`: the reference's three functions with
// their exact positional signatures (reference ext.cpp:16-20,
// integrate_primitives.h:42-139), forwarded to the C ABI of libvi_b200.so.
// Tensors become device pointers; state buffers are uint8 tensors grown by a
// resize callback, as the reference's resizeFunctional does
// (integrate_primitives.cu:54-68).  Errors raise RuntimeError.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <tuple>
#include <vector>

#include "volume_integration_b200.h"

namespace {

using torch::Tensor;

char* resize_cb(void* user, size_t n) {
  auto* t = static_cast<Tensor*>(user);
  t->resize_({(int64_t)n});
  return reinterpret_cast<char*>(t->data_ptr());
}

Tensor cuda_f32(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  return t.to(torch::kFloat32).contiguous();
}
// The kernels load one table entry's features as one vector: realign views with an odd offset.
Tensor aligned_table(const Tensor& t) {
  Tensor c = cuda_f32(t, "feature_table");
  if (reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 != 0) c = c.clone();
  return c;
}
Tensor cuda_i32(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  return t.to(torch::kInt32).contiguous();
}
void ok(int rc) { TORCH_CHECK(rc == VI_OK, "volume_integration: ", vi_last_error(), " (status ", rc, ")"); }

// Hashgrid box {lo_x, lo_y, lo_z, hi_x, hi_y, hi_z}; empty = the reference's fixed box.
const float* bounds_ptr(const std::vector<double>& hb, float* buf) {
  if (hb.empty()) return nullptr;
  TORCH_CHECK(hb.size() == 6, "hash_bounds needs 6 values (lo xyz, hi xyz), got ", hb.size());
  for (int i = 0; i < 6; i++) buf[i] = (float)hb[i];
  return buf;
}

std::tuple<int, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> integrate_primitives_ex(
    const Tensor& means3D, const Tensor& primitive_confidences, const double primitive_scale,
    const Tensor& viewmatrix, const Tensor& projmatrix, const Tensor& cam_pos, const double tan_fovx,
    const double tan_fovy, const int64_t image_height, const int64_t image_width, const double near_plane,
    const double max_distance, const Tensor& feature_table, const Tensor& resolution, const Tensor& do_hash,
    const Tensor& primes, const int64_t feature_offset, const Tensor& linear_weights, const Tensor& linear_bias,
    const int64_t stencil_genus, const int64_t grid_size, const int64_t max_primitives_per_ray,
    const double occupancy_threshold, const Tensor& bg_color, const int64_t input_feature_dim,
    const int64_t output_feature_dim, const int64_t intermediate_feature_dim, const int64_t hashgrid_levels,
    const int64_t num_output_channels, const bool debug, const std::vector<double>& hash_bounds, const int64_t flags) {
  TORCH_CHECK(means3D.dim() == 2 && means3D.size(1) == 3, "means3D must have shape (P, 3)");
  float hb[6];
  const at::cuda::CUDAGuard guard(means3D.device());
  const int P = (int)means3D.size(0), H = (int)image_height, W = (int)image_width;
  Tensor m = cuda_f32(means3D, "means3D"), c = cuda_f32(primitive_confidences, "primitive_confidences");
  Tensor vm = cuda_f32(viewmatrix, "viewmatrix"), pm = cuda_f32(projmatrix, "projmatrix");
  Tensor cp = cuda_f32(cam_pos, "cam_pos"), ft = aligned_table(feature_table);
  Tensor rs = cuda_i32(resolution, "resolution"), dh = cuda_i32(do_hash, "do_hash"), pr = cuda_i32(primes, "primes");
  Tensor lw = cuda_f32(linear_weights, "linear_weights"), lb = cuda_f32(linear_bias, "linear_bias");
  Tensor bg = cuda_f32(bg_color, "bg_color");
  TORCH_CHECK(vm.numel() >= 16 && pm.numel() >= 16, "viewmatrix/projmatrix need 16 elements");
  TORCH_CHECK(rs.numel() >= hashgrid_levels && dh.numel() >= hashgrid_levels, "resolution/do_hash need L entries");
  TORCH_CHECK(pr.numel() >= 3 && bg.numel() >= 3, "primes and bg_color need 3 entries");
  TORCH_CHECK(c.numel() == (int64_t)P * grid_size * grid_size * grid_size, "primitive_confidences must be (P, G^3)");
  auto fo = m.options();
  Tensor out_color = torch::empty({(int64_t)num_output_channels, H, W}, fo);
  Tensor out_features = torch::empty({output_feature_dim, H, W}, fo);
  Tensor visibility = torch::empty({H, W}, fo);
  auto bo = fo.dtype(torch::kUInt8);
  Tensor geom = torch::empty({0}, bo), binning = torch::empty({0}, bo), img = torch::empty({0}, bo);
  int num_rendered = 0;
  ok(vi_integrate_primitives_ex(
      resize_cb, &geom, resize_cb, &binning, resize_cb, &img, out_color.data_ptr<float>(),
      out_features.data_ptr<float>(), visibility.data_ptr<float>(), &num_rendered, P, m.data_ptr<float>(),
      c.data_ptr<float>(), (float)primitive_scale, vm.data_ptr<float>(), pm.data_ptr<float>(), cp.data_ptr<float>(),
      (float)tan_fovx, (float)tan_fovy, H, W, (float)near_plane, (float)max_distance, ft.data_ptr<float>(),
      (uint64_t)ft.numel(), rs.data_ptr<int>(), dh.data_ptr<int>(), pr.data_ptr<int>(), (int)feature_offset,
      lw.data_ptr<float>(), (uint64_t)lw.numel(), lb.data_ptr<float>(), (uint64_t)lb.numel(), (int)stencil_genus,
      (int)grid_size, (int)max_primitives_per_ray, (float)occupancy_threshold, bg.data_ptr<float>(),
      (unsigned)input_feature_dim, (unsigned)output_feature_dim, (unsigned)intermediate_feature_dim,
      (unsigned)hashgrid_levels, (unsigned)num_output_channels, debug ? 1 : 0,
      at::cuda::getCurrentCUDAStream().stream(), bounds_ptr(hash_bounds, hb), (unsigned)flags));
  return {num_rendered, out_color, out_features, visibility, geom, binning, img};
}

// The reference's 30-argument signature (integrate_primitives.h:42-62).
std::tuple<int, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> integrate_primitives(
    const Tensor& means3D, const Tensor& primitive_confidences, const double primitive_scale,
    const Tensor& viewmatrix, const Tensor& projmatrix, const Tensor& cam_pos, const double tan_fovx,
    const double tan_fovy, const int64_t image_height, const int64_t image_width, const double near_plane,
    const double max_distance, const Tensor& feature_table, const Tensor& resolution, const Tensor& do_hash,
    const Tensor& primes, const int64_t feature_offset, const Tensor& linear_weights, const Tensor& linear_bias,
    const int64_t stencil_genus, const int64_t grid_size, const int64_t max_primitives_per_ray,
    const double occupancy_threshold, const Tensor& bg_color, const int64_t input_feature_dim,
    const int64_t output_feature_dim, const int64_t intermediate_feature_dim, const int64_t hashgrid_levels,
    const int64_t num_output_channels, const bool debug) {
  return integrate_primitives_ex(means3D, primitive_confidences, primitive_scale, viewmatrix, projmatrix, cam_pos,
                                 tan_fovx, tan_fovy, image_height, image_width, near_plane, max_distance,
                                 feature_table, resolution, do_hash, primes, feature_offset, linear_weights,
                                 linear_bias, stencil_genus, grid_size, max_primitives_per_ray, occupancy_threshold,
                                 bg_color, input_feature_dim, output_feature_dim, intermediate_feature_dim,
                                 hashgrid_levels, num_output_channels, debug, {}, 0);
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> integrate_primitives_backward_ex(
    const Tensor& dL_dout_color, const Tensor& dL_dout_features, const Tensor& geomBuffer,
    const Tensor& binningBuffer, const Tensor& imgBuffer, const Tensor& means3D, const Tensor& primitive_confidences,
    const double primitive_scale, const Tensor& viewmatrix, const Tensor& projmatrix, const Tensor& cam_pos,
    const double tan_fovx, const double tan_fovy, const int64_t image_height, const int64_t image_width,
    const double near_plane, const double max_distance, const Tensor& feature_table, const Tensor& resolution,
    const Tensor& do_hash, const Tensor& primes, const int64_t feature_offset, const Tensor& linear_weights,
    const Tensor& linear_bias, const int64_t stencil_genus, const int64_t grid_size,
    const int64_t max_primitives_per_ray, const double occupancy_threshold, const Tensor& bg_color,
    const int64_t input_feature_dim, const int64_t output_feature_dim, const int64_t hashgrid_levels,
    const int64_t num_output_channels, const int64_t feature_table_size, const int64_t P, const int64_t num_rendered,
    const bool debug, const std::vector<double>& hash_bounds, const int64_t flags, const Tensor& dL_dvisibility) {
  const at::cuda::CUDAGuard guard(means3D.device());
  float hb[6];
  Tensor gv = dL_dvisibility.numel() ? cuda_f32(dL_dvisibility, "dL_dvisibility") : dL_dvisibility;
  TORCH_CHECK(!gv.numel() || gv.numel() == image_height * image_width, "dL_dvisibility must be (H, W)");
  Tensor m = cuda_f32(means3D, "means3D"), c = cuda_f32(primitive_confidences, "primitive_confidences");
  Tensor vm = cuda_f32(viewmatrix, "viewmatrix"), pm = cuda_f32(projmatrix, "projmatrix");
  Tensor cp = cuda_f32(cam_pos, "cam_pos"), ft = aligned_table(feature_table);
  Tensor rs = cuda_i32(resolution, "resolution"), dh = cuda_i32(do_hash, "do_hash"), pr = cuda_i32(primes, "primes");
  Tensor lw = cuda_f32(linear_weights, "linear_weights"), lb = cuda_f32(linear_bias, "linear_bias");
  Tensor bg = cuda_f32(bg_color, "bg_color");
  Tensor gc = cuda_f32(dL_dout_color, "dL_dout_color");
  Tensor gf = dL_dout_features.numel() ? cuda_f32(dL_dout_features, "dL_dout_features") : dL_dout_features;
  TORCH_CHECK(gc.numel() == 3 * image_height * image_width, "dL_dout_color must be (3, H, W)");
  TORCH_CHECK(gf.numel() == output_feature_dim * image_height * image_width, "dL_dout_features must be (F_out, H, W)");
  const int64_t D = hashgrid_levels * input_feature_dim, O = num_output_channels + output_feature_dim + 1;
  TORCH_CHECK(lw.numel() >= O * D && lb.numel() >= O, "linear layer needs ", O * D, " weights and ", O, " biases");
  TORCH_CHECK(c.numel() == P * grid_size * grid_size * grid_size, "primitive_confidences must be (P, G^3)");
  Tensor dmeans = torch::empty_like(m), dconf = torch::empty_like(c), dtable = torch::empty_like(ft);
  Tensor dW = torch::empty_like(lw), db = torch::empty_like(lb);
  ok(vi_integrate_primitives_backward_ex(
      dmeans.data_ptr<float>(), dconf.data_ptr<float>(), dtable.data_ptr<float>(), dW.data_ptr<float>(),
      db.data_ptr<float>(), gc.data_ptr<float>(), gf.numel() ? gf.data_ptr<float>() : nullptr,
      geomBuffer.numel() ? reinterpret_cast<char*>(geomBuffer.data_ptr()) : nullptr,
      binningBuffer.numel() ? reinterpret_cast<char*>(binningBuffer.data_ptr()) : nullptr,
      imgBuffer.numel() ? reinterpret_cast<char*>(imgBuffer.data_ptr()) : nullptr, m.data_ptr<float>(),
      c.data_ptr<float>(), (float)primitive_scale, vm.data_ptr<float>(), pm.data_ptr<float>(), cp.data_ptr<float>(),
      (float)tan_fovx, (float)tan_fovy, (int)image_height, (int)image_width, (float)near_plane, (float)max_distance,
      ft.data_ptr<float>(), rs.data_ptr<int>(), dh.data_ptr<int>(), pr.data_ptr<int>(), (int)feature_offset,
      lw.data_ptr<float>(), lb.data_ptr<float>(), (int)stencil_genus, (int)grid_size, (int)max_primitives_per_ray,
      (float)occupancy_threshold, bg.data_ptr<float>(), (unsigned)input_feature_dim, (unsigned)output_feature_dim,
      (unsigned)hashgrid_levels, (unsigned)num_output_channels, (uint64_t)feature_table_size, (int)P,
      (int)num_rendered, debug ? 1 : 0, at::cuda::getCurrentCUDAStream().stream(), bounds_ptr(hash_bounds, hb),
      (unsigned)flags, gv.numel() ? gv.data_ptr<float>() : nullptr));
  return {dmeans, dconf, dtable, dW, db};
}

// The reference's 37-argument signature (integrate_primitives.h:66-113).
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> integrate_primitives_backward(
    const Tensor& dL_dout_color, const Tensor& dL_dout_features, const Tensor& geomBuffer,
    const Tensor& binningBuffer, const Tensor& imgBuffer, const Tensor& means3D, const Tensor& primitive_confidences,
    const double primitive_scale, const Tensor& viewmatrix, const Tensor& projmatrix, const Tensor& cam_pos,
    const double tan_fovx, const double tan_fovy, const int64_t image_height, const int64_t image_width,
    const double near_plane, const double max_distance, const Tensor& feature_table, const Tensor& resolution,
    const Tensor& do_hash, const Tensor& primes, const int64_t feature_offset, const Tensor& linear_weights,
    const Tensor& linear_bias, const int64_t stencil_genus, const int64_t grid_size,
    const int64_t max_primitives_per_ray, const double occupancy_threshold, const Tensor& bg_color,
    const int64_t input_feature_dim, const int64_t output_feature_dim, const int64_t hashgrid_levels,
    const int64_t num_output_channels, const int64_t feature_table_size, const int64_t P, const int64_t num_rendered,
    const bool debug) {
  return integrate_primitives_backward_ex(
      dL_dout_color, dL_dout_features, geomBuffer, binningBuffer, imgBuffer, means3D, primitive_confidences,
      primitive_scale, viewmatrix, projmatrix, cam_pos, tan_fovx, tan_fovy, image_height, image_width, near_plane,
      max_distance, feature_table, resolution, do_hash, primes, feature_offset, linear_weights, linear_bias,
      stencil_genus, grid_size, max_primitives_per_ray, occupancy_threshold, bg_color, input_feature_dim,
      output_feature_dim, hashgrid_levels, num_output_channels, feature_table_size, P, num_rendered, debug, {}, 0,
      Tensor());
}

Tensor mark_visible(Tensor& means3D, Tensor& viewmatrix, Tensor& projmatrix) {
  const at::cuda::CUDAGuard guard(means3D.device());
  Tensor m = cuda_f32(means3D, "means3D"), vm = cuda_f32(viewmatrix, "viewmatrix");
  Tensor pm = cuda_f32(projmatrix, "projmatrix");
  Tensor present = torch::empty({m.size(0)}, m.options().dtype(torch::kBool));
  ok(vi_mark_visible((int)m.size(0), m.data_ptr<float>(), vm.data_ptr<float>(), pm.data_ptr<float>(),
                     reinterpret_cast<uint8_t*>(present.data_ptr()), at::cuda::getCurrentCUDAStream().stream()));
  return present;
}

// Views of the integer state inside the forward's buffers, in the reference's
// formats (integrator_impl.h:35-146); used by parity tests and debugging.
py::dict state_views(const Tensor& geom, const Tensor& binning, const Tensor& img, int64_t P, int64_t R, int64_t H,
                     int64_t W, int64_t K, int64_t G, int64_t Fout) {
  vi_state_layout L;
  ok(vi_get_state_layout((int)P, R, (int)H, (int)W, (int)K, (int)G, (unsigned)Fout, &L));
  auto view = [](const Tensor& buf, size_t off, int64_t n, torch::ScalarType t) {
    int64_t sz = n * (int64_t)c10::elementSize(t);
    return buf.narrow(0, (int64_t)off, sz).view(t);
  };
  const int64_t N = H * W, tiles = ((W + 15) / 16) * ((H + 15) / 16), V = G * G * G;
  py::dict d;
  if (geom.numel()) {
    d["depths"] = view(geom, L.depths, P, torch::kFloat32);
    d["radii"] = view(geom, L.radii, P, torch::kInt32);
    d["means2D"] = view(geom, L.means2D, 2 * P, torch::kFloat32).view({P, 2});
    d["tiles_touched"] = view(geom, L.tiles_touched, P, torch::kInt32);
    d["rec_cnt"] = view(geom, L.rec_cnt, P, torch::kInt32);
    d["rec_key"] = view(geom, L.rec_key, P * V, torch::kInt32);
    d["rec_props"] = view(geom, L.rec_props, P * V * L.props_stride, torch::kFloat32);
    d["status"] = view(geom, L.status, 4, torch::kInt32);
  }
  if (binning.numel() && R > 0) {
    d["sorted_tiles"] = view(binning, L.sorted_tiles, R, torch::kInt32);
    d["point_list"] = view(binning, L.point_list, R, torch::kInt32);
  }
  if (img.numel()) {
    d["ranges"] = view(img, L.ranges, 2 * tiles, torch::kInt32).view({tiles, 2});
    d["final_T"] = view(img, L.final_T, N, torch::kFloat32);
    d["n_contrib"] = view(img, L.n_contrib, N, torch::kInt32);
    d["contrib_idx"] = view(img, L.contrib_idx, N * K, torch::kInt32);
    d["delta_t"] = view(img, L.delta_t, N * K, torch::kFloat32);
    d["contrib_rec"] = view(img, L.contrib_rec, N * K, torch::kInt32);
  }
  return d;
}

// Stable sort of int64 keys (read as uint64) with int32 values over [begin_bit, end_bit).
std::tuple<Tensor, Tensor> sort_pairs(const Tensor& keys, const Tensor& vals, int64_t begin_bit, int64_t end_bit) {
  TORCH_CHECK(keys.is_cuda() && keys.scalar_type() == torch::kInt64, "keys must be CUDA int64");
  TORCH_CHECK(vals.is_cuda() && vals.scalar_type() == torch::kInt32 && vals.numel() == keys.numel(),
              "vals must be CUDA int32 of the same length");
  const at::cuda::CUDAGuard guard(keys.device());
  Tensor kin = keys.contiguous().clone(), vin = vals.contiguous().clone();
  Tensor kout = torch::empty_like(kin), vout = torch::empty_like(vin);
  size_t tb = vi_sort_pairs_temp_bytes((uint64_t)kin.numel(), (int)begin_bit, (int)end_bit);
  Tensor temp = torch::empty({(int64_t)tb}, kin.options().dtype(torch::kUInt8));
  ok(vi_sort_pairs(reinterpret_cast<uint64_t*>(kin.data_ptr()), reinterpret_cast<uint32_t*>(vin.data_ptr()),
                   reinterpret_cast<uint64_t*>(kout.data_ptr()), reinterpret_cast<uint32_t*>(vout.data_ptr()),
                   (uint64_t)kin.numel(), (int)begin_bit, (int)end_bit, temp.data_ptr(), tb,
                   at::cuda::getCurrentCUDAStream().stream()));
  return {kout, vout};
}

}  // namespace

// ---- Gaussian-attribute front end (extension; no counterpart in the reference) ----

Tensor aligned16(const Tensor& t) {
  Tensor c = cuda_f32(t, "tensor");
  if (reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 != 0) c = c.clone();
  return c;
}

// The camera position by value (a device tensor costs a blocking copy).
std::vector<float> host3(const Tensor& t) {
  Tensor h = t.detach().to(torch::kCPU, torch::kFloat32).contiguous().view({-1});
  TORCH_CHECK(h.numel() == 3, "campos must hold 3 values");
  return {h[0].item<float>(), h[1].item<float>(), h[2].item<float>()};
}

// (radii, means2D, depths, cov3D, conic_opacity, rgb, clamped, tiles_touched)
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> preprocess_gaussians(
    const Tensor& means3D, const Tensor& scales, const Tensor& rotations, const Tensor& opacities, const Tensor& shs,
    int64_t sh_degree, double scale_modifier, const Tensor& viewmatrix, const Tensor& projmatrix, const Tensor& campos,
    int64_t image_width, int64_t image_height, double tan_fovx, double tan_fovy, double near_plane) {
  const at::cuda::OptionalCUDAGuard guard(means3D.device());
  Tensor m = cuda_f32(means3D, "means3D"), sc = cuda_f32(scales, "scales"), q = aligned16(rotations);
  Tensor op = cuda_f32(opacities, "opacities"), sh = cuda_f32(shs, "shs");
  Tensor vm = cuda_f32(viewmatrix, "viewmatrix"), pm = cuda_f32(projmatrix, "projmatrix");
  const int64_t P = m.size(0);
  TORCH_CHECK(m.dim() == 2 && m.size(1) == 3 && sc.sizes() == m.sizes(), "means3D and scales must be [P, 3]");
  TORCH_CHECK(q.dim() == 2 && q.size(0) == P && q.size(1) == 4, "rotations must be [P, 4]");
  TORCH_CHECK(op.numel() == P, "opacities must hold P values");
  TORCH_CHECK(sh.dim() == 3 && sh.size(0) == P && sh.size(2) == 3, "shs must be [P, M, 3]");
  const std::vector<float> cp = host3(campos);
  auto f32 = m.options();
  Tensor radii = torch::empty({P}, f32.dtype(torch::kInt32));
  Tensor means2D = torch::empty({P, 2}, f32), depths = torch::empty({P}, f32), cov3D = torch::empty({P, 6}, f32);
  Tensor conic = torch::empty({P, 4}, f32), rgb = torch::empty({P, 3}, f32);
  Tensor clamped = torch::empty({P, 3}, f32.dtype(torch::kUInt8));
  Tensor tiles = torch::empty({P}, f32.dtype(torch::kInt32));
  ok(vi_preprocess_gaussians((int)P, (int)sh_degree, (int)sh.size(1), m.data_ptr<float>(), sc.data_ptr<float>(),
                             q.data_ptr<float>(), op.data_ptr<float>(), sh.data_ptr<float>(), (float)scale_modifier,
                             vm.data_ptr<float>(), pm.data_ptr<float>(), cp.data(), (int)image_width,
                             (int)image_height, (float)tan_fovx, (float)tan_fovy, (float)near_plane,
                             radii.data_ptr<int>(), means2D.data_ptr<float>(), depths.data_ptr<float>(),
                             cov3D.data_ptr<float>(), conic.data_ptr<float>(), rgb.data_ptr<float>(),
                             reinterpret_cast<uint8_t*>(clamped.data_ptr()),
                             reinterpret_cast<uint32_t*>(tiles.data_ptr()), at::cuda::getCurrentCUDAStream().stream()));
  return {radii, means2D, depths, cov3D, conic, rgb, clamped, tiles};
}

// (dL/dmeans3D, dL/dscales, dL/drotations, dL/dshs)
std::tuple<Tensor, Tensor, Tensor, Tensor> preprocess_gaussians_backward(
    const Tensor& means3D, const Tensor& scales, const Tensor& rotations, const Tensor& shs, int64_t sh_degree,
    double scale_modifier, const Tensor& viewmatrix, const Tensor& projmatrix, const Tensor& campos,
    int64_t image_width, int64_t image_height, double tan_fovx, double tan_fovy, double near_plane,
    const Tensor& radii, const Tensor& clamped, const Tensor& dL_dmeans2D, const Tensor& dL_ddepths,
    const Tensor& dL_dcov3D, const Tensor& dL_dconic_opacity, const Tensor& dL_drgb) {
  const at::cuda::OptionalCUDAGuard guard(means3D.device());
  Tensor m = cuda_f32(means3D, "means3D"), sc = cuda_f32(scales, "scales"), q = aligned16(rotations);
  Tensor sh = cuda_f32(shs, "shs");
  Tensor vm = cuda_f32(viewmatrix, "viewmatrix"), pm = cuda_f32(projmatrix, "projmatrix");
  Tensor rd = cuda_i32(radii, "radii");
  TORCH_CHECK(clamped.is_cuda() && clamped.scalar_type() == torch::kUInt8, "clamped must be a CUDA uint8 tensor");
  Tensor cl = clamped.contiguous();
  const int64_t P = m.size(0);
  Tensor g2 = cuda_f32(dL_dmeans2D, "dL_dmeans2D"), gd = cuda_f32(dL_ddepths, "dL_ddepths");
  Tensor gcov = cuda_f32(dL_dcov3D, "dL_dcov3D"), gco = cuda_f32(dL_dconic_opacity, "dL_dconic_opacity");
  Tensor grgb = cuda_f32(dL_drgb, "dL_drgb");
  TORCH_CHECK(g2.numel() == 2 * P && gd.numel() == P && gcov.numel() == 6 * P && gco.numel() == 4 * P &&
                  grgb.numel() == 3 * P && rd.numel() == P && cl.numel() == 3 * P,
              "gradient shapes do not match P");
  const std::vector<float> cp = host3(campos);
  Tensor dm = torch::empty({P, 3}, m.options()), ds = torch::empty({P, 3}, m.options());
  Tensor dq = torch::empty({P, 4}, m.options()), dsh = torch::empty_like(sh);
  ok(vi_preprocess_gaussians_backward(
      (int)P, (int)sh_degree, (int)sh.size(1), m.data_ptr<float>(), sc.data_ptr<float>(), q.data_ptr<float>(),
      sh.data_ptr<float>(), (float)scale_modifier, vm.data_ptr<float>(), pm.data_ptr<float>(), cp.data(),
      (int)image_width, (int)image_height, (float)tan_fovx, (float)tan_fovy, (float)near_plane, rd.data_ptr<int>(),
      reinterpret_cast<const uint8_t*>(cl.data_ptr()), g2.data_ptr<float>(), gd.data_ptr<float>(),
      gcov.data_ptr<float>(), gco.data_ptr<float>(), grgb.data_ptr<float>(), dm.data_ptr<float>(),
      ds.data_ptr<float>(), dq.data_ptr<float>(), dsh.data_ptr<float>(), at::cuda::getCurrentCUDAStream().stream()));
  return {dm, ds, dq, dsh};
}

// (point_list [R] int32, tile ids [R] int32, ranges [tiles, 2] int32)
std::tuple<Tensor, Tensor, Tensor> bin_gaussians(const Tensor& radii, const Tensor& means2D, const Tensor& depths,
                                                 const Tensor& tiles_touched, int64_t image_width,
                                                 int64_t image_height) {
  const at::cuda::OptionalCUDAGuard guard(radii.device());
  Tensor rd = cuda_i32(radii, "radii"), m2 = cuda_f32(means2D, "means2D"), dp = cuda_f32(depths, "depths");
  Tensor tt = cuda_i32(tiles_touched, "tiles_touched");
  const int64_t P = rd.numel();
  TORCH_CHECK(m2.numel() == 2 * P && dp.numel() == P && tt.numel() == P, "binning inputs must describe P Gaussians");
  const int64_t R = P ? tt.sum(torch::kInt64).item<int64_t>() : 0;  // buffer sizing; the scan re-checks it
  const int64_t tiles = ((image_width + 15) / 16) * ((image_height + 15) / 16);
  auto i32 = rd.options();
  Tensor point_list = torch::empty({R}, i32), tile_ids = torch::empty({R}, i32);
  Tensor ranges = torch::empty({tiles, 2}, i32);
  const uint64_t nbytes = vi_bin_gaussians_scratch_bytes((int)P, (uint64_t)R, (int)image_width, (int)image_height);
  TORCH_CHECK(nbytes > 0, "volume_integration: bad binning sizes");
  Tensor scratch = torch::empty({(int64_t)nbytes + 256}, rd.options().dtype(torch::kUInt8));
  char* base = reinterpret_cast<char*>(scratch.data_ptr());
  char* al = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(base) + 255) & ~uintptr_t(255));
  ok(vi_bin_gaussians((int)P, (int)image_width, (int)image_height, rd.data_ptr<int>(), m2.data_ptr<float>(),
                      dp.data_ptr<float>(), reinterpret_cast<const uint32_t*>(tt.data_ptr()), (uint64_t)R, al, nbytes,
                      R ? reinterpret_cast<uint32_t*>(point_list.data_ptr()) : nullptr,
                      R ? reinterpret_cast<uint32_t*>(tile_ids.data_ptr()) : nullptr,
                      reinterpret_cast<uint32_t*>(ranges.data_ptr()), at::cuda::getCurrentCUDAStream().stream()));
  return {point_list, tile_ids, ranges};
}

// ---- per-pixel heads ----
namespace {

int head_dtype(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return VI_F32;
    case torch::kFloat16: return VI_F16;
    case torch::kBFloat16: return VI_BF16;
    default: TORCH_CHECK(false, name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
  }
}
// What every tensor of a heads call must share with x.
void head_like(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == x.device(), name, " must be on ", x.device(), ", got ", t.device());
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " must be ", x.scalar_type(), ", got ", t.scalar_type());
}
vi_matrix head_matrix(const Tensor& t) { return {t.data_ptr(), t.size(0), t.size(1), t.stride(0), t.stride(1)}; }
// The 2D matrix of an optional tensor; nullptr when there is none.
struct OptMatrix {
  vi_matrix m{};
  bool on;
  OptMatrix(const c10::optional<Tensor>& t, const Tensor& x, const char* name) : on(t.has_value()) {
    if (!on) return;
    head_like(*t, x, name);
    TORCH_CHECK(t->dim() == 2, name, " must be 2D");
    m = head_matrix(*t);
  }
  const vi_matrix* get() const { return on ? &m : nullptr; }
};
void head_check(const Tensor& x, const Tensor& weight) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  TORCH_CHECK(x.dim() == 2 && weight.dim() == 2, "x and weight must be 2D");
  head_like(weight, x, "weight");
}
Tensor head_bias(const c10::optional<Tensor>& bias, const Tensor& x, const Tensor& weight) {
  if (!bias.has_value()) return {};
  head_like(*bias, x, "bias");
  TORCH_CHECK(bias->dim() == 1 && bias->size(0) == weight.size(0), "bias must be [", weight.size(0), "]");
  return bias->contiguous();
}
Tensor head_target(const Tensor& target, const Tensor& x) {
  TORCH_CHECK(target.is_cuda() && target.device() == x.device(), "target must be on ", x.device());
  TORCH_CHECK(target.scalar_type() == torch::kInt64 && target.dim() == 1 && target.size(0) == x.size(0),
              "target must be int64 [", x.size(0), "]");
  return target.contiguous();
}
void* head_ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// A new [rows, cols] in x's memory order: columns contiguous unless x is [K, rows] in memory.
Tensor head_result(const Tensor& x, int64_t rows, int64_t cols) {
  const bool image = x.stride(0) == 1 && x.stride(1) != 1;
  return image ? torch::empty({cols, rows}, x.options()).t() : torch::empty({rows, cols}, x.options());
}
Tensor head_scratch(uint64_t bytes, const Tensor& x) {
  TORCH_CHECK(bytes > 0, "volume_integration: ", vi_last_error());
  if (bytes <= 256) return {};  // nothing but the query's constant: the call takes none
  return torch::empty({(int64_t)bytes}, x.options().dtype(torch::kUInt8));
}

// (y, act' or None)
std::tuple<Tensor, c10::optional<Tensor>> linear_act_forward(const Tensor& x, const Tensor& weight,
                                                             const c10::optional<Tensor>& bias,
                                                             const c10::optional<Tensor>& residual, int64_t activation,
                                                             bool backward_follows) {
  head_check(x, weight);
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dt = head_dtype(x, "x");
  const Tensor b = head_bias(bias, x, weight);
  const OptMatrix r(residual, x, "residual");
  const vi_matrix mx = head_matrix(x), mw = head_matrix(weight);
  Tensor y = head_result(x, x.size(0), weight.size(0));
  c10::optional<Tensor> dact;
  vi_matrix my = head_matrix(y), md{};
  const bool want_dact = backward_follows && vi_linear_act_keeps_dact(dt, (int)activation, &mx, &mw);
  if (want_dact) {
    dact = torch::empty_like(y);
    md = head_matrix(*dact);
  }
  const uint64_t n = vi_linear_act_forward_scratch_bytes(dt, (int)activation, &mx, &mw, head_ptr(b), r.get(), &my,
                                                         want_dact ? &md : nullptr);
  Tensor scratch = head_scratch(n, x);
  ok(vi_linear_act_forward(dt, (int)activation, &mx, &mw, head_ptr(b), r.get(), &my, want_dact ? &md : nullptr,
                           head_ptr(scratch), n, at::cuda::getCurrentCUDAStream().stream()));
  return {y, dact};
}

using Grads = std::tuple<c10::optional<Tensor>, c10::optional<Tensor>, c10::optional<Tensor>>;

// Gradient tensors of x, weight and bias, those that are wanted.
struct GradTensors {
  c10::optional<Tensor> dx, dw, db;
  vi_matrix mx{}, mw{};
  GradTensors(const Tensor& x, const Tensor& weight, bool need_x, bool need_w, bool need_b) {
    if (need_x) dx = head_result(x, x.size(0), x.size(1)), mx = head_matrix(*dx);
    if (need_w) dw = torch::empty({weight.size(0), weight.size(1)}, x.options()), mw = head_matrix(*dw);
    if (need_b) db = torch::empty({weight.size(0)}, x.options());
  }
  const vi_matrix* x() const { return dx.has_value() ? &mx : nullptr; }
  const vi_matrix* w() const { return dw.has_value() ? &mw : nullptr; }
  void* b() const { return db.has_value() ? db->data_ptr() : nullptr; }
};

// (dx, dweight, dbias), None where not wanted
Grads linear_act_backward(const Tensor& dy, const c10::optional<Tensor>& dact, const Tensor& x, const Tensor& weight,
                          const c10::optional<Tensor>& bias, int64_t activation, bool need_x, bool need_w, bool need_b) {
  head_check(x, weight);
  head_like(dy, x, "dy");
  TORCH_CHECK(dy.dim() == 2, "dy must be 2D");
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dt = head_dtype(x, "x");
  const Tensor b = head_bias(bias, x, weight);
  const OptMatrix d(dact, x, "dact");
  const vi_matrix mdy = head_matrix(dy), mx = head_matrix(x), mw = head_matrix(weight);
  GradTensors g(x, weight, need_x, need_w, need_b);
  const uint64_t n = vi_linear_act_backward_scratch_bytes(dt, (int)activation, &mdy, d.get(), &mx, &mw, head_ptr(b),
                                                          g.x(), g.w(), g.b());
  Tensor scratch = head_scratch(n, x);
  ok(vi_linear_act_backward(dt, (int)activation, &mdy, d.get(), &mx, &mw, head_ptr(b), g.x(), g.w(), g.b(),
                            head_ptr(scratch), n, at::cuda::getCurrentCUDAStream().stream()));
  return {g.dx, g.dw, g.db};
}

// (loss, lse)
std::tuple<Tensor, Tensor> linear_ce_forward(const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias,
                                             const Tensor& target, int64_t ignore_index, int64_t reduction) {
  head_check(x, weight);
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dt = head_dtype(x, "x");
  const Tensor b = head_bias(bias, x, weight), t = head_target(target, x);
  const vi_matrix mx = head_matrix(x), mw = head_matrix(weight);
  const auto f32 = x.options().dtype(torch::kFloat32);
  Tensor loss = reduction == VI_REDUCE_NONE ? torch::empty({x.size(0)}, f32) : torch::empty({}, f32);
  Tensor lse = torch::empty({3, x.size(0)}, f32);
  const uint64_t n = vi_linear_ce_forward_scratch_bytes(dt, &mx, &mw, head_ptr(b));
  Tensor scratch = head_scratch(n, x);
  ok(vi_linear_ce_forward(dt, &mx, &mw, head_ptr(b), t.data_ptr<int64_t>(), ignore_index, (int)reduction,
                          loss.data_ptr<float>(), lse.data_ptr<float>(), head_ptr(scratch), n,
                          at::cuda::getCurrentCUDAStream().stream()));
  return {loss, lse};
}

// (dx, dweight, dbias), None where not wanted
Grads linear_ce_backward(const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias, const Tensor& target,
                         int64_t ignore_index, int64_t reduction, const Tensor& lse, const Tensor& dloss, bool need_x,
                         bool need_w, bool need_b) {
  head_check(x, weight);
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dt = head_dtype(x, "x");
  const Tensor b = head_bias(bias, x, weight), t = head_target(target, x);
  Tensor l = cuda_f32(lse, "lse"), dl = cuda_f32(dloss, "dloss");
  TORCH_CHECK(l.numel() == 3 * x.size(0), "lse must be [3, ", x.size(0), "]");
  TORCH_CHECK(dl.numel() == (reduction == VI_REDUCE_NONE ? x.size(0) : 1), "dloss does not fit the reduction");
  const vi_matrix mx = head_matrix(x), mw = head_matrix(weight);
  GradTensors g(x, weight, need_x, need_w, need_b);
  const uint64_t n = vi_linear_ce_backward_scratch_bytes(dt, &mx, &mw, head_ptr(b), g.x(), g.w(), g.b());
  Tensor scratch = head_scratch(n, x);
  ok(vi_linear_ce_backward(dt, &mx, &mw, head_ptr(b), t.data_ptr<int64_t>(), ignore_index, (int)reduction,
                           l.data_ptr<float>(), dl.data_ptr<float>(), g.x(), g.w(), g.b(), head_ptr(scratch), n,
                           at::cuda::getCurrentCUDAStream().stream()));
  return {g.dx, g.dw, g.db};
}

// The heads as differentiable functions.  In C++, so that a step on a few rows does not spend its
// time in the interpreter; a second derivative raises, as torch's once_differentiable does.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void differentiate_once(variable_list& grads) {
  if (!torch::GradMode::is_enabled()) return;
  variable_list fake;
  std::vector<size_t> at;
  for (size_t i = 0; i < grads.size(); i++) {
    if (!grads[i].defined()) continue;
    Tensor t = grads[i].detach();
    t.set_requires_grad(true);
    fake.push_back(t);
    at.push_back(i);
  }
  if (fake.empty()) return;
  auto fn = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)fake.size());
  variable_list out = (*fn)(std::move(fake));
  for (size_t i = 0; i < at.size(); i++) grads[at[i]] = out[i];
}
c10::optional<Tensor> optional_of(const Tensor& t) { return t.defined() ? c10::optional<Tensor>(t) : c10::nullopt; }
// The kernels carry no tangents, and an input with one need not require a gradient: it would be dropped without a word.
template <class... T>
void no_tangents(const char* what, const T&... ts) {
  const auto has = [](const c10::optional<Tensor>& t) { return t.has_value() && t->defined() && t->_fw_grad(0).defined(); };
  TORCH_CHECK(!(has(ts) || ...), what, ": forward-mode differentiation is not supported");
}
bool capturing() { return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None; }
// Whether a leaf's gradient would be handed to the default stream, because an eager graph on it still lives.  Under a
// capture autograd would then make that stream wait for the captured one, which CUDA forbids, and
// the error ends the process: the backward refuses before.
bool bound_to_default_stream(const c10::optional<Tensor>& t) {
  if (!t.has_value() || !t->defined() || !t->requires_grad() || !t->is_leaf()) return false;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
  const auto s = node ? node->stream() : std::nullopt;
  return s.has_value() && s->device_type() == c10::DeviceType::CUDA &&
         c10::cuda::CUDAStream(c10::cuda::CUDAStream::UNCHECKED, *s).stream() == nullptr;
}
// The inputs of which that holds, bit i for the i-th; 0 outside a capture.
template <class... T>
int64_t bound_to_default_stream(const T&... ts) {
  if (!capturing()) return 0;
  int64_t mask = 0, bit = 1;
  ((mask |= bound_to_default_stream(c10::optional<Tensor>(ts)) ? bit : 0, bit *= 2), ...);
  return mask;
}
void check_capture(AutogradContext* ctx, std::initializer_list<bool> needed, const char* what) {
  int64_t mask = 0, bit = 1;
  for (const bool n : needed) mask |= n ? bit : 0, bit *= 2;
  TORCH_CHECK(!(ctx->saved_data["default_stream"].toInt() & mask) || !capturing(), what,
              ": captured, while an earlier result of the same leaves, computed on the default stream, is still alive; let go of "
              "it (del) before the capture, or compute it on another stream");
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const c10::optional<Tensor>& t) { return t.has_value() && t->requires_grad(); }

struct LinearAct : torch::autograd::Function<LinearAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias,
                        const c10::optional<Tensor>& residual, int64_t activation) {
    // act' is kept rather than z, so the backward needs no transcendental; relu's is read off the result
    head_check(x, weight);
    const vi_matrix mx = head_matrix(x), mw = head_matrix(weight);
    const bool from_y = activation == VI_ACT_RELU && !residual.has_value() &&
                        vi_linear_act_keeps_dact(head_dtype(x, "x"), VI_ACT_RELU, &mx, &mw);
    auto [y, dact] = linear_act_forward(x, weight, bias, residual, activation,
                                        !from_y && (wants_grad(x) || wants_grad(weight) || wants_grad(bias)));
    if (from_y) dact = y;
    ctx->save_for_backward({x, weight, bias.value_or(Tensor()), dact.value_or(Tensor())});
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["default_stream"] = bound_to_default_stream(x, weight, bias, residual);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dys) {
    no_tangents("linear_act backward", dys[0]);
    const variable_list saved = ctx->get_saved_variables();
    const bool has_b = ctx->saved_data["bias"].toBool(), has_r = ctx->saved_data["residual"].toBool();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nb = has_b && ctx->needs_input_grad(2);
    const bool nr = has_r && ctx->needs_input_grad(has_b ? 3 : 2);
    check_capture(ctx, {nx, nw, nb, nr}, "linear_act backward");
    variable_list out(5);
    if (nx || nw || nb) {
      auto [dx, dw, db] = linear_act_backward(dys[0], optional_of(saved[3]), saved[0], saved[1], optional_of(saved[2]),
                                              ctx->saved_data["activation"].toInt(), nx, nw, nb);
      if (nx) out[0] = *dx;
      if (nw) out[1] = *dw;
      if (nb) out[2] = *db;
    }
    differentiate_once(out);
    if (nr) out[3] = dys[0];
    return out;
  }
};

Tensor linear_act(const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias,
                  const c10::optional<Tensor>& residual, int64_t activation) {
  no_tangents("linear_act", x, weight, bias, residual);
  if (torch::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias) || wants_grad(residual)))
    return LinearAct::apply(x, weight, bias, residual, activation);
  return std::get<0>(linear_act_forward(x, weight, bias, residual, activation, false));
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias,
                        const Tensor& target, int64_t ignore_index, int64_t reduction) {
    auto [loss, lse] = linear_ce_forward(x, weight, bias, target, ignore_index, reduction);
    ctx->save_for_backward({x, weight, bias.value_or(Tensor()), target, lse});
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["ignore"] = ignore_index;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["default_stream"] = bound_to_default_stream(x, weight, bias);
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dloss) {
    no_tangents("linear_cross_entropy backward", dloss[0]);
    const variable_list saved = ctx->get_saved_variables();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1);
    const bool nb = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
    check_capture(ctx, {nx, nw, nb}, "linear_cross_entropy backward");
    variable_list out(6);
    if (nx || nw || nb) {
      auto [dx, dw, db] =
          linear_ce_backward(saved[0], saved[1], optional_of(saved[2]), saved[3], ctx->saved_data["ignore"].toInt(),
                             ctx->saved_data["reduction"].toInt(), saved[4], dloss[0], nx, nw, nb);
      if (nx) out[0] = *dx;
      if (nw) out[1] = *dw;
      if (nb) out[2] = *db;
    }
    differentiate_once(out);
    return out;
  }
};

Tensor linear_cross_entropy(const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias,
                            const Tensor& target, int64_t ignore_index, int64_t reduction) {
  no_tangents("linear_cross_entropy", x, weight, bias);
  if (torch::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias)))
    return LinearCrossEntropy::apply(x, weight, bias, target, ignore_index, reduction);
  return std::get<0>(linear_ce_forward(x, weight, bias, target, ignore_index, reduction));
}

// A vector of K elements that belongs to x's columns, contiguous.
Tensor norm_vector(const c10::optional<Tensor>& v, const Tensor& x, const char* name) {
  if (!v.has_value()) return {};
  head_like(*v, x, name);
  TORCH_CHECK(v->dim() == 1 && v->size(0) == x.size(1), name, " must be [", x.size(1), "]");
  return v->contiguous();
}

// (y, stats or None)
std::tuple<Tensor, c10::optional<Tensor>> layer_norm_forward(const Tensor& x, const c10::optional<Tensor>& weight,
                                                             const c10::optional<Tensor>& bias, double eps, bool backward_follows) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "x must be a 2D CUDA tensor");
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dt = head_dtype(x, "x");
  const Tensor w = norm_vector(weight, x, "weight"), b = norm_vector(bias, x, "bias");
  Tensor y = head_result(x, x.size(0), x.size(1));
  c10::optional<Tensor> stats;
  if (backward_follows) stats = torch::empty({3, x.size(0)}, x.options().dtype(torch::kFloat32));
  const vi_matrix mx = head_matrix(x), my = head_matrix(y);
  ok(vi_layer_norm_forward(dt, &mx, head_ptr(w), head_ptr(b), (float)eps, &my, stats ? stats->data_ptr<float>() : nullptr,
                           at::cuda::getCurrentCUDAStream().stream()));
  return {y, stats};
}

// (dx, dweight, dbias), None where not wanted
Grads layer_norm_backward(const Tensor& dy, const Tensor& x, const c10::optional<Tensor>& weight, const Tensor& stats, bool need_x,
                          bool need_w, bool need_b) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "x must be a 2D CUDA tensor");
  head_like(dy, x, "dy");
  TORCH_CHECK(dy.dim() == 2 && dy.size(0) == x.size(0) && dy.size(1) == x.size(1), "dy must have x's shape");
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dt = head_dtype(x, "x");
  const Tensor w = norm_vector(weight, x, "weight"), st = cuda_f32(stats, "stats");
  TORCH_CHECK(st.numel() == 3 * x.size(0) && st.device() == x.device(), "stats must be [3, ", x.size(0), "] on ", x.device());
  const vi_matrix mdy = head_matrix(dy), mx = head_matrix(x);
  c10::optional<Tensor> dx, dw, db;
  vi_matrix mdx{};
  if (need_x) dx = head_result(x, x.size(0), x.size(1)), mdx = head_matrix(*dx);
  if (need_w) dw = torch::empty({x.size(1)}, x.options());
  if (need_b) db = torch::empty({x.size(1)}, x.options());
  const vi_matrix* pdx = need_x ? &mdx : nullptr;
  void *pdw = need_w ? dw->data_ptr() : nullptr, *pdb = need_b ? db->data_ptr() : nullptr;
  const uint64_t n = vi_layer_norm_backward_scratch_bytes(dt, &mdy, &mx, head_ptr(w), pdx, pdw, pdb);
  Tensor scratch = head_scratch(n, x);
  ok(vi_layer_norm_backward(dt, &mdy, &mx, head_ptr(w), st.data_ptr<float>(), pdx, pdw, pdb, head_ptr(scratch), n,
                            at::cuda::getCurrentCUDAStream().stream()));
  return {dx, dw, db};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const c10::optional<Tensor>& weight,
                        const c10::optional<Tensor>& bias, double eps) {
    auto [y, stats] = layer_norm_forward(x, weight, bias, eps, true);
    ctx->save_for_backward({x, weight.value_or(Tensor()), *stats});
    ctx->saved_data["weight"] = weight.has_value();
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["default_stream"] = bound_to_default_stream(x, weight, bias);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dys) {
    no_tangents("layer_norm backward", dys[0]);
    const variable_list saved = ctx->get_saved_variables();
    const bool has_w = ctx->saved_data["weight"].toBool(), has_b = ctx->saved_data["bias"].toBool();
    const bool nx = ctx->needs_input_grad(0), nw = has_w && ctx->needs_input_grad(1);
    const bool nb = has_b && ctx->needs_input_grad(has_w ? 2 : 1);
    check_capture(ctx, {nx, nw, nb}, "layer_norm backward");
    variable_list out(4);
    if (nx || nw || nb) {
      auto [dx, dw, db] = layer_norm_backward(dys[0], saved[0], optional_of(saved[1]), saved[2], nx, nw, nb);
      if (nx) out[0] = *dx;
      if (nw) out[1] = *dw;
      if (nb) out[2] = *db;
    }
    differentiate_once(out);
    return out;
  }
};

Tensor layer_norm(const Tensor& x, const c10::optional<Tensor>& weight, const c10::optional<Tensor>& bias, double eps) {
  no_tangents("layer_norm", x, weight, bias);
  if (torch::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias)))
    return LayerNorm::apply(x, weight, bias, eps);
  return std::get<0>(layer_norm_forward(x, weight, bias, eps, false));
}

// (q [M, K] int8 with rows a multiple of 16 bytes apart, scale [M])
std::tuple<Tensor, Tensor> quantize_rows(const Tensor& x) {
  no_tangents("quantize_rows", x);
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "x must be a 2D CUDA tensor");
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dt = head_dtype(x, "x");
  const int64_t K = x.size(1);
  Tensor q = torch::empty({x.size(0), (K + 15) / 16 * 16}, x.options().dtype(torch::kInt8)).slice(1, 0, K);
  Tensor scale = torch::empty({x.size(0)}, x.options().dtype(torch::kFloat32));
  const vi_matrix mx = head_matrix(x), mq = head_matrix(q);
  ok(vi_quantize_rows(dt, &mx, &mq, scale.data_ptr<float>(), at::cuda::getCurrentCUDAStream().stream()));
  return {q, scale};
}

// x of `dtype`, or int8 with x_scale
Tensor linear_act_int8(const Tensor& x, const c10::optional<Tensor>& x_scale, const Tensor& weight, const Tensor& weight_scale,
                       const c10::optional<Tensor>& bias, const c10::optional<Tensor>& residual, int64_t activation,
                       c10::ScalarType dtype) {
  no_tangents("linear_act_int8", x, x_scale, weight_scale, bias, residual);
  TORCH_CHECK(!torch::GradMode::is_enabled() || !(wants_grad(x) || wants_grad(x_scale) || wants_grad(weight_scale) ||
                                                  wants_grad(bias) || wants_grad(residual)),
              "linear_act_int8 has no backward: call it under torch.no_grad(), or with detached tensors");
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && weight.dim() == 2, "x and weight must be 2D CUDA tensors");
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const auto scale_of = [&](const Tensor& s, int64_t n, const char* name) {
    TORCH_CHECK(s.device() == x.device() && s.scalar_type() == torch::kFloat32 && s.dim() == 1 && s.size(0) == n, name,
                " must be float32 [", n, "] on ", x.device());
    return s.contiguous();
  };
  TORCH_CHECK(weight.device() == x.device() && weight.scalar_type() == torch::kInt8, "weight must be int8 on ", x.device());
  TORCH_CHECK(x.scalar_type() == (x_scale.has_value() ? torch::kInt8 : dtype), "x must be ", x_scale.has_value() ? torch::kInt8 : dtype);
  const Tensor ws = scale_of(weight_scale, weight.size(0), "weight's scale");
  const Tensor xs = x_scale.has_value() ? scale_of(*x_scale, x.size(0), "x's scale") : Tensor();
  const auto options = x.options().dtype(dtype);
  Tensor y = x.stride(0) == 1 && x.stride(1) != 1 ? torch::empty({weight.size(0), x.size(0)}, options).t()
                                                  : torch::empty({x.size(0), weight.size(0)}, options);
  const int dt = head_dtype(y, "the result");
  const Tensor b = head_bias(bias, y, weight);
  const OptMatrix r(residual, y, "residual");
  const vi_matrix mx = head_matrix(x), mw = head_matrix(weight), my = head_matrix(y);
  const float *pxs = xs.defined() ? xs.data_ptr<float>() : nullptr, *pws = ws.data_ptr<float>();
  const uint64_t n = vi_linear_act_int8_scratch_bytes(dt, (int)activation, &mx, pxs, &mw, pws, head_ptr(b), r.get(), &my);
  Tensor scratch = head_scratch(n, x);
  ok(vi_linear_act_int8(dt, (int)activation, &mx, pxs, &mw, pws, head_ptr(b), r.get(), &my, head_ptr(scratch), n,
                        at::cuda::getCurrentCUDAStream().stream()));
  return y;
}

// A setting is its tensor, where that is given, else its number.
Tensor sample_labels(const Tensor& logits, const Tensor& u, double temperature, const c10::optional<Tensor>& temperatures,
                     int64_t top_k, const c10::optional<Tensor>& top_ks, double top_p, const c10::optional<Tensor>& top_ps,
                     double min_p, const c10::optional<Tensor>& min_ps) {
  no_tangents("sample_labels", logits, u, temperatures, top_ps, min_ps);
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, "logits must be a 2D CUDA tensor");
  const at::cuda::OptionalCUDAGuard guard(logits.device());
  const int dt = head_dtype(logits, "logits");
  const auto rows_of = [&](const c10::optional<Tensor>& t, c10::ScalarType type, const char* name) {
    if (!t.has_value()) return Tensor();
    TORCH_CHECK(t->device() == logits.device() && t->scalar_type() == type && t->dim() == 1 && t->size(0) == logits.size(0), name,
                " must be ", type, " [", logits.size(0), "] on ", logits.device());
    return t->contiguous();
  };
  const Tensor v = rows_of(u, torch::kFloat32, "u"), t = rows_of(temperatures, torch::kFloat32, "temperature"),
               k = rows_of(top_ks, torch::kInt64, "top_k"), p = rows_of(top_ps, torch::kFloat32, "top_p"),
               m = rows_of(min_ps, torch::kFloat32, "min_p");
  const auto f32 = [](const Tensor& x) { return x.defined() ? x.data_ptr<float>() : nullptr; };
  const vi_sampling s{temperature, top_p, min_p, top_k, f32(t), k.defined() ? k.data_ptr<int64_t>() : nullptr, f32(p), f32(m)};
  Tensor label = torch::empty({logits.size(0)}, logits.options().dtype(torch::kInt64));
  const vi_matrix mz = head_matrix(logits);
  const uint64_t n = vi_sample_labels_scratch_bytes(dt, &mz, &s);
  Tensor scratch = head_scratch(n, logits);
  ok(vi_sample_labels(dt, &mz, v.data_ptr<float>(), &s, label.data_ptr<int64_t>(), head_ptr(scratch), n,
                      at::cuda::getCurrentCUDAStream().stream()));
  return label;
}

// The heads' status word of a device (0 = no wait gave up).
int64_t heads_status(int64_t device, bool reset) {
  const at::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  uint32_t word = 0;
  ok(vi_heads_status(&word, reset ? 1 : 0, at::cuda::getCurrentCUDAStream().stream()));
  return word;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("integrate_primitives", &integrate_primitives, "Integrate Primitives CUDA forward");
  m.def("integrate_primitives_backward", &integrate_primitives_backward, "Integrate Primitives CUDA backward");
  m.def("integrate_primitives_ex", &integrate_primitives_ex,
        "integrate_primitives plus a hashgrid box (6 floats, or [] for the reference's box) and flags "
        "(1 = exact gradients)");
  m.def("integrate_primitives_backward_ex", &integrate_primitives_backward_ex,
        "integrate_primitives_backward plus the hashgrid box, flags and dL/dvisibility (empty = none)");
  m.attr("FLAG_EXACT_GRADIENTS") = (int64_t)VI_FLAG_EXACT_GRADIENTS;
  m.def("mark_visible", &mark_visible, "Mark Visible Primitives CUDA");
  m.def("preprocess_gaussians", &preprocess_gaussians, "Gaussian-attribute preprocess (extension)");
  m.def("preprocess_gaussians_backward", &preprocess_gaussians_backward,
        "Exact derivative of the Gaussian-attribute preprocess (extension)");
  m.def("bin_gaussians", &bin_gaussians, "Tile binning of projected Gaussians (extension)");
  m.def("linear_act", &linear_act, "act(x W^T + b) + residual, differentiable (extension)");
  m.def("linear_cross_entropy", &linear_cross_entropy, "Cross entropy of a linear classifier, differentiable (extension)");
  m.def("linear_act_forward", &linear_act_forward, "act(x W^T + b) + residual (extension)");
  m.def("linear_act_backward", &linear_act_backward, "Gradients of linear_act_forward (extension)");
  m.def("linear_ce_forward", &linear_ce_forward, "Cross entropy of a linear classifier (extension)");
  m.def("linear_ce_backward", &linear_ce_backward, "Gradients of linear_ce_forward (extension)");
  m.def("layer_norm", &layer_norm, "Layer norm of rows, differentiable (extension)");
  m.def("layer_norm_forward", &layer_norm_forward, "Layer norm of rows (extension)");
  m.def("layer_norm_backward", &layer_norm_backward, "Gradients of layer_norm_forward (extension)");
  m.def("quantize_rows", &quantize_rows, "Rows in 8-bit integers with a scale each (extension)");
  m.def("linear_act_int8", &linear_act_int8, "act(x W^T + b) + residual with 8-bit integer products (extension)");
  m.def("sample_labels", &sample_labels, "Labels drawn from rows of logits (extension)");
  m.def("heads_status", &heads_status, "Status word of the heads' kernels on a device (extension)");
  m.def("state_views", &state_views, "Integer state of a forward call in the reference's formats");
  m.def("sort_pairs", &sort_pairs, "Stable radix sort of (uint64 key, uint32 value) pairs");
  m.def("sort_end_bit", [](int64_t tiles) { return vi_sort_end_bit((uint32_t)tiles); });
  m.def("kernel_launches", []() { return (uint64_t)vi_kernel_launches(); });
  m.def("profile_enable", [](bool on) { ok(vi_profile_enable(on ? 1 : 0)); });
  m.def("profile_read", [](bool reset) {
    double ms[8];
    uint64_t calls[8];
    ok(vi_profile_read(ms, calls, 8, reset ? 1 : 0));
    static const char* names[8] = {"preprocess", "depth_sort", "offsets", "features",
                                   "binning", "render", "bwd_pixel", "bwd_prim"};
    py::dict d;
    for (int i = 0; i < 8; i++) d[names[i]] = py::make_tuple(ms[i], calls[i]);
    return d;
  });
}
