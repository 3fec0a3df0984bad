// gnr_torch.cpp -- the PyTorch-ROCm C++ binding of libgnr.so ("PyTorch-ROCm C++/HIP extension").
//
// Host code only: it validates torch tensors (TORCH_CHECK -> Python exceptions, so the reference's
// `try: ... except: continue` around a batch, trainer/gazenerf_trainer.py:576-582, keeps working), sets the device
// guard, takes the CURRENT HIP stream of the tensors' device, allocates outputs and workspaces as torch tensors
// (the caching allocator owns every byte) and calls the C ABI of include/gnr.h.  No kernels live here, and nothing
// here computes: a missing / failing library call is an error, never a fallback.
//
// Python surface (gazenerf_amd/render.py picks this binding when the module is built, else the ctypes one):
//   render_fwd(...) -> [feat_0, bg_alpha_0, (depth_0), (weights_0), feat_1, ..., workspace]
//   render_bwd(...) -> [dR, dT, dshape, dgaze, dappea, 24 gradients per weight set ...]
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <string>
#include <vector>

#include "../../include/gnr.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

void check_f32(const Tensor& t, const char* name, const c10::Device& dev) {
    TORCH_CHECK(t.defined(), name, " must be a tensor");
    TORCH_CHECK(t.device() == dev, name, " must live on ", dev, " (the render op has no CPU path), got ", t.device());
    TORCH_CHECK(t.scalar_type() == at::kFloat, name, " must be float32, got ", t.scalar_type());
}

struct Problem {
    GnrProblem c = GNR_INIT_PROBLEM;   // zeroed + struct_size stamped (size handshake)
    std::vector<Tensor> keep;          // contiguous versions the pointers refer to
    int64_t B = 0, n_r = 0, n_p = 0;
    c10::Device dev{c10::kCPU};
};

Problem make_problem(const Tensor& xy, const Tensor& R, const Tensor& T, const Tensor& Kinv, const Tensor& shape_code,
                     const Tensor& gaze, const Tensor& appea_code, const OptTensor& t_rand, const OptTensor& z_edges,
                     int64_t n_samples, double world_z1, double world_z2, int64_t hidden, int64_t feat_nc,
                     bool edges_follow_T, int64_t vd_dims = 0, const OptTensor& ray_bias0 = c10::nullopt,
                     const OptTensor& ray_bias1 = c10::nullopt) {
    Problem p;
    TORCH_CHECK(xy.defined() && xy.is_cuda(), "batch_xy must live on a CUDA/ROCm device (the render op has no CPU path)");
    p.dev = xy.device();
    check_f32(xy, "batch_xy", p.dev);
    TORCH_CHECK(xy.dim() == 3 && xy.size(1) == 2, "batch_xy must be [B,2,N_r], got ", xy.sizes());
    p.B = xy.size(0); p.n_r = xy.size(2); p.n_p = n_samples;
    auto want = [&](const Tensor& t, const char* name, std::vector<int64_t> shape) {
        check_f32(t, name, p.dev);
        TORCH_CHECK(t.sizes() == at::IntArrayRef(shape), name, " must have shape ", at::IntArrayRef(shape), ", got ", t.sizes());
    };
    want(R, "R", {p.B, 3, 3});
    want(T, "T", {p.B, 3, 1});
    want(Kinv, "Kinv", {p.B, 3, 3});
    for (auto pr : {std::make_pair(&shape_code, "shape_code"), std::make_pair(&gaze, "gaze"), std::make_pair(&appea_code, "appea_code")}) {
        check_f32(*pr.first, pr.second, p.dev);
        TORCH_CHECK(pr.first->dim() == 2 && pr.first->size(0) == p.B, pr.second, " must be [", p.B, ", dims], got ", pr.first->sizes());
    }
    if (t_rand) want(*t_rand, "t_rand", {p.B, p.n_r, n_samples + 1});
    if (z_edges) want(*z_edges, "z_edges", {p.B, p.n_r, n_samples + 1});
    auto keep = [&](const Tensor& t) { p.keep.push_back(t.contiguous()); return p.keep.back().data_ptr<float>(); };
    GnrProblem& c = p.c;
    c.batch = (int32_t)p.B; c.n_rays = (int32_t)p.n_r; c.n_samples = (int32_t)n_samples;
    c.hidden = (int32_t)hidden; c.feat_nc = (int32_t)feat_nc;
    c.shape_dims = (int32_t)shape_code.size(1); c.gaze_dims = (int32_t)gaze.size(1); c.appea_dims = (int32_t)appea_code.size(1);
    c.world_z1 = (float)world_z1; c.world_z2 = (float)world_z2;
    c.xy = keep(xy); c.R = keep(R); c.T = keep(T); c.Kinv = keep(Kinv);
    c.shape_code = keep(shape_code); c.gaze = keep(gaze); c.appea_code = keep(appea_code);
    c.t_rand = t_rand ? keep(*t_rand) : nullptr;
    c.z_edges = z_edges ? keep(*z_edges) : nullptr;
    c.edges_follow_T = (edges_follow_T && z_edges) ? 1 : 0;
    // view-direction option (include/gnr.h): skipped weight columns + per-ray bias of RGB_layer_1 per weight set
    TORCH_CHECK(vd_dims >= 0, "vd_dims must be >= 0");
    c.vd_dims = (int32_t)vd_dims;
    const OptTensor* rb[2] = {&ray_bias0, &ray_bias1};
    for (int s = 0; s < 2; ++s)
        if (*rb[s]) {
            want(**rb[s], "ray_bias", {p.B, p.n_r, hidden / 2});
            c.ray_bias[s] = keep(**rb[s]);
        }
    return p;
}

// 24 tensors of one MLPforNeRF in PARAM_ORDER (FeaExt_module_0..7 weight/bias, density, RGB_layer_0..2); Conv2d
// [out,in,1,1] memory == row-major [out,in].  Returns contiguous 2-D/1-D views kept alive in `keep`.
void fill_weights(const std::vector<Tensor>& params, const Problem& p, int64_t hidden, int64_t feat_nc, const char* tag,
                  std::vector<Tensor>& keep, GnrWeights* w) {
    TORCH_CHECK(params.size() == 24, tag, ": expected 24 parameter tensors, got ", params.size());
    const int64_t vp = 63 + p.c.shape_dims + p.c.gaze_dims, ap = p.c.vd_dims + p.c.appea_dims;
    auto mat = [&](int i, int64_t rows, int64_t cols) {
        Tensor t = params[i];
        check_f32(t, tag, p.dev);
        if (t.dim() == 4) {
            TORCH_CHECK(t.size(2) == 1 && t.size(3) == 1, tag, "[", i, "]: only 1x1 kernels");
            t = t.reshape({t.size(0), t.size(1)});
        }
        TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, tag, "[", i, "] must have shape [", rows, ", ", cols,
                    "], got ", params[i].sizes());
        keep.push_back(t.contiguous());
        return (const float*)keep.back().data_ptr<float>();
    };
    auto vec = [&](int i, int64_t n) {
        const Tensor& t = params[i];
        check_f32(t, tag, p.dev);
        TORCH_CHECK(t.dim() == 1 && t.size(0) == n, tag, "[", i, "] must have shape [", n, "], got ", t.sizes());
        keep.push_back(t.contiguous());
        return (const float*)keep.back().data_ptr<float>();
    };
    for (int l = 0; l < 8; ++l) {
        const int64_t cin = l == 0 ? vp : (l == 5 ? hidden + vp : hidden);
        w->fea_w[l] = mat(2 * l, hidden, cin);
        w->fea_b[l] = vec(2 * l + 1, hidden);
    }
    w->density_w = mat(16, 1, hidden);
    w->density_b = vec(17, 1);
    w->rgb_w[0] = mat(18, hidden, hidden);          w->rgb_b[0] = vec(19, hidden);
    w->rgb_w[1] = mat(20, hidden / 2, hidden + ap); w->rgb_b[1] = vec(21, hidden / 2);
    w->rgb_w[2] = mat(22, feat_nc, hidden / 2);     w->rgb_b[2] = vec(23, feat_nc);
}

void check_rc(int rc) { TORCH_CHECK(rc == 0, gnr_last_error()); }

Tensor alloc_ws(size_t bytes, const c10::Device& dev) {
    return at::empty({(int64_t)(bytes < 256 ? 256 : bytes)}, at::TensorOptions().dtype(at::kByte).device(dev));
}

std::vector<Tensor> render_fwd(const Tensor& xy, const Tensor& R, const Tensor& T, const Tensor& Kinv, const Tensor& shape_code,
                               const Tensor& gaze, const Tensor& appea_code, const OptTensor& t_rand, const OptTensor& z_edges,
                               const std::vector<Tensor>& face, const std::vector<Tensor>& eyes, int64_t n_samples, double world_z1,
                               double world_z2, int64_t hidden, int64_t feat_nc, bool save, bool want_depth, bool want_weights,
                               bool bf16x3, bool edges_follow_T, const OptTensor& ws_in, bool weights_packed, int64_t vd_dims,
                               const OptTensor& ray_bias0, const OptTensor& ray_bias1) {
    Problem p = make_problem(xy, R, T, Kinv, shape_code, gaze, appea_code, t_rand, z_edges, n_samples, world_z1, world_z2, hidden,
                             feat_nc, edges_follow_T, vd_dims, ray_bias0, ray_bias1);
    const c10::DeviceGuard guard(p.dev);
    const int n_streams = eyes.empty() ? 1 : 2;
    const size_t nbytes = gnr_workspace_bytes(&p.c, n_streams, save ? GNR_WS_FWD_SAVE : GNR_WS_FWD);
    // a caller-owned workspace (render.PackedWeightCache) whose packed weights may still be current
    TORCH_CHECK(!weights_packed || (ws_in && !save), "weights_packed needs the caller's workspace and an inference call");
    if (ws_in) {
        TORCH_CHECK(ws_in->is_cuda() && ws_in->device() == p.dev && ws_in->scalar_type() == at::kByte && ws_in->is_contiguous() &&
                    (size_t)ws_in->numel() >= nbytes, "workspace must be a contiguous uint8 tensor of >= ", nbytes, " bytes on ", p.dev);
    }
    p.c.weights_packed = weights_packed ? 1 : 0;
    TORCH_CHECK(nbytes != 0, gnr_last_error());
    std::vector<Tensor> keep;
    GnrWeights w[2]{};
    fill_weights(face, p, hidden, feat_nc, "stream0", keep, &w[0]);
    if (n_streams > 1) fill_weights(eyes, p, hidden, feat_nc, "stream1", keep, &w[1]);
    Tensor ws = ws_in ? *ws_in : alloc_ws(nbytes, p.dev);
    const auto opt = at::TensorOptions().dtype(at::kFloat).device(p.dev);
    GnrOutputs out{};
    std::vector<Tensor> res;
    for (int s = 0; s < n_streams; ++s) {
        Tensor feat = at::empty({p.B, feat_nc, p.n_r}, opt), bga = at::empty({p.B, 1, p.n_r}, opt);
        out.feat[s] = feat.data_ptr<float>();
        out.bg_alpha[s] = bga.data_ptr<float>();
        res.push_back(feat);
        res.push_back(bga);
        if (want_depth) {
            Tensor d = at::empty({p.B, 1, p.n_r}, opt);
            out.depth[s] = d.data_ptr<float>();
            res.push_back(d);
        }
        if (want_weights) {
            Tensor wt = at::empty({p.B, 1, p.n_r, p.n_p}, opt);
            out.weights[s] = wt.data_ptr<float>();
            res.push_back(wt);
        }
    }
    void* stream = (void*)c10::hip::getCurrentHIPStream(p.dev.index()).stream();
    auto fn = bf16x3 ? gnr_fwd_bf16x3 : gnr_fwd;
    check_rc(fn(&p.c, &w[0], n_streams > 1 ? &w[1] : nullptr, &out, save ? 1 : 0, ws.data_ptr(), (size_t)ws.numel(), stream));
    res.push_back(ws);
    return res;
}

std::vector<Tensor> render_bwd(const Tensor& xy, const Tensor& R, const Tensor& T, const Tensor& Kinv, const Tensor& shape_code,
                               const Tensor& gaze, const Tensor& appea_code, const OptTensor& t_rand, const OptTensor& z_edges,
                               const std::vector<Tensor>& face, const std::vector<Tensor>& eyes,
                               const std::vector<OptTensor>& d_feat, const std::vector<OptTensor>& d_bg_alpha, const Tensor& saved_ws,
                               int64_t n_samples, double world_z1, double world_z2, int64_t hidden, int64_t feat_nc, bool bf16x3,
                               bool edges_follow_T, int64_t vd_dims, const OptTensor& ray_bias0, const OptTensor& ray_bias1) {
    Problem p = make_problem(xy, R, T, Kinv, shape_code, gaze, appea_code, t_rand, z_edges, n_samples, world_z1, world_z2, hidden,
                             feat_nc, edges_follow_T, vd_dims, ray_bias0, ray_bias1);
    const c10::DeviceGuard guard(p.dev);
    const int n_streams = eyes.empty() ? 1 : 2;
    TORCH_CHECK((int)d_feat.size() == n_streams && (int)d_bg_alpha.size() == n_streams, "one (d_feat, d_bg_alpha) pair per weight set");
    TORCH_CHECK(saved_ws.defined() && saved_ws.device() == p.dev && saved_ws.scalar_type() == at::kByte,
                "saved workspace must be the uint8 tensor render_fwd(save=True) returned");
    std::vector<Tensor> keep;
    GnrWeights w[2]{};
    fill_weights(face, p, hidden, feat_nc, "stream0", keep, &w[0]);
    if (n_streams > 1) fill_weights(eyes, p, hidden, feat_nc, "stream1", keep, &w[1]);
    GnrOutputGrads dout{};
    for (int s = 0; s < n_streams; ++s) {
        if (d_feat[s]) {
            check_f32(*d_feat[s], "d_feat", p.dev);
            TORCH_CHECK(d_feat[s]->sizes() == at::IntArrayRef({p.B, feat_nc, p.n_r}), "d_feat must be [B,feat_nc,N_r]");
            keep.push_back(d_feat[s]->contiguous());
            dout.feat[s] = keep.back().data_ptr<float>();
        }
        if (d_bg_alpha[s]) {
            check_f32(*d_bg_alpha[s], "d_bg_alpha", p.dev);
            TORCH_CHECK(d_bg_alpha[s]->sizes() == at::IntArrayRef({p.B, 1, p.n_r}), "d_bg_alpha must be [B,1,N_r]");
            keep.push_back(d_bg_alpha[s]->contiguous());
            dout.bg_alpha[s] = keep.back().data_ptr<float>();
        }
    }
    const auto opt = at::TensorOptions().dtype(at::kFloat).device(p.dev);
    std::vector<Tensor> res = {at::empty({p.B, 3, 3}, opt), at::empty({p.B, 3, 1}, opt), at::empty({p.B, p.c.shape_dims}, opt),
                               at::empty({p.B, p.c.gaze_dims}, opt), at::empty({p.B, p.c.appea_dims}, opt)};
    GnrInputGrads din{};
    din.R = res[0].data_ptr<float>(); din.T = res[1].data_ptr<float>(); din.shape_code = res[2].data_ptr<float>();
    din.gaze = res[3].data_ptr<float>(); din.appea_code = res[4].data_ptr<float>();
    GnrWeightGrads dw[2]{};
    for (int s = 0; s < n_streams; ++s) {
        const std::vector<Tensor>& src = s == 0 ? face : eyes;
        float* ptr[24];
        for (int i = 0; i < 24; ++i) {
            Tensor g = at::empty(src[i].sizes(), opt);           // same shape as the parameter ([out,in,1,1] stays 4-D)
            ptr[i] = g.data_ptr<float>();
            res.push_back(g);
        }
        for (int l = 0; l < 8; ++l) { dw[s].fea_w[l] = ptr[2 * l]; dw[s].fea_b[l] = ptr[2 * l + 1]; }
        dw[s].density_w = ptr[16]; dw[s].density_b = ptr[17];
        for (int l = 0; l < 3; ++l) { dw[s].rgb_w[l] = ptr[18 + 2 * l]; dw[s].rgb_b[l] = ptr[19 + 2 * l]; }
    }
    // d ray_bias per weight set, appended after the parameter gradients (an undefined tensor == None where absent)
    Tensor grb[2];
    for (int s = 0; s < n_streams; ++s)
        if (p.c.ray_bias[s]) {
            grb[s] = at::empty({p.B, p.n_r, hidden / 2}, opt);
            din.ray_bias[s] = grb[s].data_ptr<float>();
        }
    const size_t sbytes = gnr_workspace_bytes(&p.c, n_streams, GNR_WS_BWD);
    TORCH_CHECK(sbytes != 0, gnr_last_error());
    Tensor scratch = alloc_ws(sbytes, p.dev);
    void* stream = (void*)c10::hip::getCurrentHIPStream(p.dev.index()).stream();
    auto fn = bf16x3 ? gnr_bwd_bf16x3 : gnr_bwd;
    check_rc(fn(&p.c, &w[0], n_streams > 1 ? &w[1] : nullptr, &dout, &din, &dw[0], n_streams > 1 ? &dw[1] : nullptr,
                saved_ws.data_ptr(), (size_t)saved_ws.numel(), scratch.data_ptr(), (size_t)scratch.numel(), stream));
    res.push_back(grb[0]);
    res.push_back(grb[1]);
    return res;
}

int64_t saved_workspace_bytes(int64_t batch, int64_t n_rays, int64_t n_samples, int64_t hidden, int64_t feat_nc, int64_t n_streams) {
    GnrProblem c = GNR_INIT_PROBLEM;
    c.batch = (int32_t)batch; c.n_rays = (int32_t)n_rays; c.n_samples = (int32_t)n_samples; c.hidden = (int32_t)hidden;
    c.feat_nc = (int32_t)feat_nc;
    static const float dummy = 0.0f;                 // sizes only: pointers are checked for NULL, never dereferenced
    c.xy = c.R = c.T = c.Kinv = &dummy;
    const size_t n = gnr_workspace_bytes(&c, (int)n_streams, GNR_WS_FWD_SAVE);
    TORCH_CHECK(n != 0, gnr_last_error());
    return (int64_t)n;
}


// ---- 8-bit rows (gazenerf_amd/int8.py documents the operators) ------------------------------------------------------------------
int type_id(at::ScalarType t, const char* name) {
    switch (t) {
        case at::kFloat: return GNR_F32;
        case at::kBFloat16: return GNR_BF16;
        case at::kHalf: return GNR_F16;
        default: TORCH_CHECK(false, name, " must be float32, bfloat16 or float16, got ", t);
    }
    return -1;
}
at::ScalarType type_of(int64_t id) {
    TORCH_CHECK(id == GNR_F32 || id == GNR_BF16 || id == GNR_F16, "unknown type id ", id);
    return id == GNR_F32 ? at::kFloat : (id == GNR_BF16 ? at::kBFloat16 : at::kHalf);
}
void check_on(const Tensor& t, const char* name, at::ScalarType type, int64_t dims, const c10::Device& dev) {
    TORCH_CHECK(t.defined() && t.device() == dev, name, " must live on ", dev);
    TORCH_CHECK(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
    TORCH_CHECK(dims < 0 || t.dim() == dims, name, " must have ", dims, " dimensions, got shape ", t.sizes());
}
void check_cuda(const Tensor& t, const char* name) {
    TORCH_CHECK(t.defined() && t.is_cuda(), name, " must live on a CUDA/ROCm device (the 8-bit operators have no CPU path)");
}
int64_t row_pitch(int64_t k) { return (k + 63) / 64 * 64; }
Tensor empty_rows(int64_t b, int64_t n, int64_t k, const c10::Device& dev) {
    Tensor t = at::empty({b, n, row_pitch(k)}, at::TensorOptions().dtype(at::kChar).device(dev));
    return t.slice(2, 0, k);
}
// [B, C, ...] -> [B, C, P], [..., K] -> [b, n, K]: views, or copies where the strides need them
Tensor maps3(const Tensor& t) {
    TORCH_CHECK(t.dim() >= 3, "maps must be [B, C, ...], got ", t.sizes());
    Tensor m = t;
    if (t.dim() != 3) {
        int64_t pix = 1;
        for (int64_t d = 2; d < t.dim(); ++d) pix *= t.size(d);
        m = t.reshape({t.size(0), t.size(1), pix});
    }
    return m.stride(2) == 1 || m.size(2) <= 1 ? m : m.contiguous();
}
Tensor rows3(const Tensor& t) {
    TORCH_CHECK(t.dim() >= 1, "rows must be [..., K]");
    const int64_t k = t.size(-1);
    Tensor m = t;
    if (t.dim() == 2) {
        m = t.unsqueeze(0);
    } else if (t.dim() != 3) {
        int64_t n = 1;
        for (int64_t d = 0; d + 1 < t.dim(); ++d) n *= t.size(d);
        m = t.reshape({1, n, k});
    }
    return m.stride(2) == 1 || k <= 1 ? m : m.contiguous();
}
int64_t stride_or(const Tensor& t, int64_t d, int64_t other) { return t.size(d) > 1 ? t.stride(d) : other; }
// Rows [..., K] as (entries, rows of an entry) with two strides; `keep` holds the tensor the pointer belongs to.  2-D and 3-D tensors are
// described as they are (a view costs half a microsecond), others through a reshape.
struct RowsIn {
    Tensor keep;
    int64_t b = 1, n = 1, k = 0, sb = 0, sn = 0;
};
RowsIn rows_in(const Tensor& t) {
    RowsIn r;
    r.keep = t.dim() == 2 || t.dim() == 3 ? t : rows3(t);
    const int64_t d = r.keep.dim();
    r.k = r.keep.size(d - 1);
    if (r.k > 1 && r.keep.stride(d - 1) != 1) r.keep = r.keep.contiguous();
    r.n = r.keep.size(d - 2);
    r.sn = r.keep.stride(d - 2);
    if (d == 3) { r.b = r.keep.size(0); r.sb = r.keep.stride(0); }
    return r;
}
// 8-bit rows as a product reads them: on 16-byte boundaries, readable to the next multiple of 16
RowsIn rows8_in(const Tensor& t) {
    RowsIn r = rows_in(t);
    const int64_t k16 = (r.k + 15) / 16 * 16;
    if (r.n <= 1) r.sn = k16;
    if (r.b <= 1) r.sb = 0;
    bool ok = r.sn % 16 == 0 && r.sn >= k16 && r.sb % 16 == 0 && (uintptr_t)r.keep.data_ptr() % 16 == 0;
    if (ok && r.b > 0 && r.n > 0)
        ok = r.keep.storage_offset() + (r.b - 1) * r.sb + (r.n - 1) * r.sn + k16 <= (int64_t)r.keep.storage().nbytes();
    if (!ok) {
        Tensor out = empty_rows(r.b, r.n, r.k, t.device());
        out.copy_(r.keep.dim() == 3 ? r.keep : r.keep.unsqueeze(0));
        r.keep = out; r.sn = row_pitch(r.k); r.sb = r.sn * r.n;
    }
    return r;
}
void* stream_of(const c10::Device& dev) { return (void*)c10::hip::getCurrentHIPStream(dev.index()).stream(); }

GnrRowsProblem rows_problem(const Tensor& x3, bool cf, const Tensor& q, const Tensor& scale) {
    GnrRowsProblem p = GNR_INIT_ROWS_PROBLEM;
    p.dtype = type_id(x3.scalar_type(), "x"); p.channels_first = cf;
    TORCH_CHECK(x3.size(0) <= INT32_MAX && x3.size(cf ? 1 : 2) <= INT32_MAX, "too many maps or channels: ", x3.sizes());
    p.batch = (int32_t)x3.size(0); p.channels = (int32_t)x3.size(cf ? 1 : 2); p.n_pix = x3.size(cf ? 2 : 1);
    p.x = x3.data_ptr(); p.x_batch = x3.stride(0); p.x_stride = x3.stride(1);
    p.q = (int8_t*)q.data_ptr(); p.q_batch = q.stride(0); p.q_pitch = stride_or(q, 1, row_pitch(q.size(2)));
    p.scale = scale.data_ptr<float>(); p.scale_batch = scale.stride(0);
    return p;
}

std::vector<Tensor> quantize_rows(const Tensor& x, bool cf) {
    check_cuda(x, "x");
    type_id(x.scalar_type(), "x");
    const c10::DeviceGuard guard(x.device());
    const Tensor x3 = cf ? maps3(x) : rows3(x);
    const int64_t b = x3.size(0), n = x3.size(cf ? 2 : 1), k = x3.size(cf ? 1 : 2);
    TORCH_CHECK(k >= 1, "x has no channels: ", x.sizes());
    Tensor q = empty_rows(b, n, k, x.device()), scale = at::empty({b, n}, at::TensorOptions().dtype(at::kFloat).device(x.device()));
    if (x3.numel() != 0) {
        const GnrRowsProblem p = rows_problem(x3, cf, q, scale);
        check_rc(gnr_quantize_rows(&p, stream_of(x.device())));
    }
    if (!cf && x.dim() != 3) {
        std::vector<int64_t> lead(x.sizes().begin(), x.sizes().end() - 1), shape(x.sizes().begin(), x.sizes().end()), strides(shape.size(), 1);
        int64_t s = row_pitch(k);
        for (size_t d = lead.size(); d-- > 0;) { strides[d] = s; s *= lead[d]; }
        q = q.as_strided(shape, strides);
        scale = scale.view(lead);
    }
    return {q, scale};
}

void check_cache(const Tensor& q, const Tensor& scale, const Tensor& slots) {
    check_cuda(q, "q");
    check_on(q, "q", at::kChar, 3, q.device());
    check_on(scale, "scale", at::kFloat, 2, q.device());
    check_on(slots, "slots", at::kLong, 1, q.device());
    const int64_t n = q.size(0), p = q.size(1), c = q.size(2);
    TORCH_CHECK(n >= 1 && p >= 1 && c >= 1, "the cache is empty: q ", q.sizes());
    TORCH_CHECK(scale.size(0) == n && scale.size(1) == p, "scale must have shape [", n, ", ", p, "], got ", scale.sizes());
    TORCH_CHECK((c == 1 || q.stride(2) == 1) && (p == 1 || q.stride(1) >= c) && (n == 1 || q.stride(0) >= (p - 1) * q.stride(1) + c),
                "q must have its channels contiguous and its rows apart, got strides ", q.strides());
    TORCH_CHECK((p == 1 || scale.stride(1) == 1) && (n == 1 || scale.stride(0) >= p),
                "scale must have its pixels contiguous and its slots apart, got strides ", scale.strides());
}

void write_featmaps(const Tensor& q, const Tensor& scale, const Tensor& slots, const Tensor& maps) {
    check_cache(q, scale, slots);
    TORCH_CHECK(maps.defined() && maps.device() == q.device(), "maps must live on ", q.device());
    type_id(maps.scalar_type(), "maps");
    const c10::DeviceGuard guard(q.device());
    const Tensor m = maps3(maps), sl = slots.contiguous();
    TORCH_CHECK(m.size(0) == sl.size(0) && m.size(1) == q.size(2) && m.size(2) == q.size(1), "maps must be [", sl.size(0), ", ", q.size(2),
                ", ...] with ", q.size(1), " pixels, got ", maps.sizes());
    if (m.numel() == 0) return;
    GnrRowsProblem p = rows_problem(m, true, q, scale);
    p.slots = sl.data_ptr<int64_t>(); p.n_slots = q.size(0);
    check_rc(gnr_quantize_rows(&p, stream_of(q.device())));
}

Tensor read_featmaps(const Tensor& q, const Tensor& scale, const Tensor& slots, int64_t out_type) {
    check_cache(q, scale, slots);
    const c10::DeviceGuard guard(q.device());
    const Tensor sl = slots.contiguous();
    Tensor out = at::empty({sl.size(0), q.size(2), q.size(1)}, at::TensorOptions().dtype(type_of(out_type)).device(q.device()));
    if (out.numel() == 0) return out;
    GnrRowsProblem p = rows_problem(out, true, q, scale);
    p.slots = sl.data_ptr<int64_t>(); p.n_slots = q.size(0);
    check_rc(gnr_read_rows(&p, stream_of(q.device())));
    return out;
}

Tensor int8_linear(const Tensor& x, const Tensor& w_q, const Tensor& w_scale, const OptTensor& bias, const OptTensor& x_scale,
                   const OptTensor& slots, bool leaky, bool cf, int64_t out_type) {
    check_cuda(x, "x");
    const c10::Device dev = x.device();
    const c10::DeviceGuard guard(dev);
    const bool rows8 = x.scalar_type() == at::kChar;
    check_on(w_q, "w_q", at::kChar, 2, dev);
    check_on(w_scale, "w_scale", at::kFloat, 1, dev);
    const int64_t o = w_q.size(0), k = w_q.size(1);
    TORCH_CHECK(o >= 1 && k >= 1 && o <= 1 << 27 && k <= GNR_INT8_MAX_K, "w_q has a shape the product cannot take: ", w_q.sizes());
    TORCH_CHECK(w_scale.size(0) == o, "w_scale must have shape [", o, "], got ", w_scale.sizes());
    GnrInt8Problem p = GNR_INIT_INT8_PROBLEM;
    p.x_type = rows8 ? GNR_I8 : type_id(x.scalar_type(), "x");
    const at::ScalarType yt = type_of(out_type);
    p.y_type = (int32_t)out_type; p.leaky = leaky; p.y_channels_first = cf; p.k = (int32_t)k; p.o = (int32_t)o;
    const RowsIn w = rows8_in(w_q);
    const Tensor ws_c = w_scale.contiguous();
    Tensor b_c, xs, sl;
    RowsIn xr;
    if (bias) {
        check_on(*bias, "bias", at::kFloat, 1, dev);
        TORCH_CHECK(bias->size(0) == o, "bias must have shape [", o, "], got ", bias->sizes());
        b_c = bias->contiguous();
    }
    int64_t b, n;
    std::vector<int64_t> shape;
    if (rows8) {
        TORCH_CHECK(x_scale, "8-bit x needs its x_scale");
        TORCH_CHECK(x.dim() >= 1 && x.size(-1) == k, "x has another number of channels than w_q: ", x.sizes(), ", ", w_q.sizes());
        TORCH_CHECK((!slots && !cf) || x.dim() == 3, "with slots or channels_first, 8-bit x must be [n, P, K], got ", x.sizes());
        check_on(*x_scale, "x_scale", at::kFloat, x.dim() - 1, dev);
        TORCH_CHECK(x_scale->sizes() == x.sizes().slice(0, x.dim() - 1), "x_scale must have the shape of x without its channels, got ",
                    x_scale->sizes());
        xr = rows8_in(x);
        b = xr.b; n = xr.n;
        xs = x.dim() == 3 || x.dim() == 2 ? *x_scale : x_scale->reshape({b, n});
        if (n > 1 && xs.stride(xs.dim() - 1) != 1) xs = xs.contiguous();
        p.x_scale = xs.data_ptr<float>(); p.x_scale_batch = xs.dim() == 2 ? xs.stride(0) : 0;
        p.x_batch = xr.sb; p.x_stride = xr.sn;
        if (slots) {
            check_on(*slots, "slots", at::kLong, 1, dev);
            TORCH_CHECK(b >= 1, "slots are given but x is empty: ", x.sizes());
            sl = slots->contiguous();
            p.slots = sl.data_ptr<int64_t>(); p.n_slots = b;
            b = sl.size(0);
        }
        if (cf) shape = {b, o, n};
        else if (slots) shape = {b, n, o};
    } else {
        TORCH_CHECK(!x_scale && !slots, "x_scale and slots go with 8-bit x; floating x is quantised by the call");
        if (cf) {
            xr.keep = maps3(x);
            xr.b = xr.keep.size(0); xr.k = xr.keep.size(1); xr.n = xr.keep.size(2); xr.sb = xr.keep.stride(0); xr.sn = xr.keep.stride(1);
        } else {
            TORCH_CHECK(x.dim() >= 1, "rows must be [..., K]");
            xr = rows_in(x);
            // entries that stand one behind the other are one: which kernel takes them goes by their number, not by how they are counted
            if (xr.b > 1 && (xr.n == 1 || xr.sb == xr.n * xr.sn)) {
                if (xr.n == 1) xr.sn = xr.sb;
                xr.n *= xr.b;
                xr.b = 1;
            }
        }
        b = xr.b; n = xr.n;
        TORCH_CHECK(xr.k == k, "x has another number of channels than w_q: ", x.sizes(), ", ", w_q.sizes());
        p.x_channels_first = cf; p.x_batch = xr.sb; p.x_stride = xr.sn;
        if (cf) {
            shape = x.sizes().vec();
            shape[1] = o;
        }
    }
    if (shape.empty()) {
        shape = x.sizes().vec();
        shape.back() = o;
    }
    Tensor y = at::empty(shape, at::TensorOptions().dtype(yt).device(dev));
    if (y.numel() == 0) return y;
    TORCH_CHECK(b <= INT32_MAX, "too many entries: ", b);
    p.batch = (int32_t)b; p.n_pix = n; p.x = xr.keep.data_ptr();
    p.w = (const int8_t*)w.keep.data_ptr(); p.w_pitch = w.sn; p.w_scale = ws_c.data_ptr<float>();
    p.bias = bias ? b_c.data_ptr<float>() : nullptr;
    p.y = y.data_ptr();
    const size_t need = gnr_int8_linear_workspace_bytes(&p);
    TORCH_CHECK(need != 0, gnr_last_error());
    Tensor ws;
    if (need > 256) ws = alloc_ws(need, dev);                  // 256: none is used
    check_rc(gnr_int8_linear(&p, need > 256 ? ws.data_ptr() : nullptr, need > 256 ? (size_t)ws.numel() : 0, stream_of(dev)));
    return y;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "PyTorch-ROCm C++ binding of libgnr.so (GazeNeRF volumetric hot path on MI355X)";
    m.def("abi_version", []() { return gnr_abi_version(); });
#ifndef GNR_SOURCE_HASH
#define GNR_SOURCE_HASH "unknown"
#endif
    m.def("source_hash", []() { return std::string(GNR_SOURCE_HASH); }, "hash of csrc/ + include/gnr.h this binding was built from");
    m.def("build_info", []() { return std::string(gnr_build_info()); }, "gnr_build_info() of the libgnr.so it is linked to");
    m.def("render_fwd", &render_fwd, "gnr_fwd / gnr_fwd_bf16x3 on the current HIP stream");
    m.def("render_bwd", &render_bwd, "gnr_bwd / gnr_bwd_bf16x3 on the current HIP stream");
    m.def("quantize_rows", &quantize_rows, "gnr_quantize_rows on the current HIP stream -> [q, scale]");
    m.def("write_featmaps", &write_featmaps, "gnr_quantize_rows into the slots of a cache");
    m.def("read_featmaps", &read_featmaps, "gnr_read_rows from the slots of a cache");
    m.def("int8_linear", &int8_linear, "gnr_int8_linear on the current HIP stream");
    m.def("saved_workspace_bytes", &saved_workspace_bytes, "bytes of saved activations for a training forward of this size");
}
