"""8-bit rows (gazenerf_amd.int8): quantise, cache write / read, the integer product, and a run of them together, against plain
implementations in 64 bits.

What has ONE answer is compared bit for bit: the whole steps q, the scales (a quotient of two fp32 numbers formed in 64 bits and
rounded to 32 is the correctly rounded one, 53 >= 2 * 24 + 2) and the values read back.  The product's sum is exact; its epilogue
rounds in fp32 (u = 2^-24): the sum to fp32, two scalings, the bias, the slope 0.2 and its product -- six roundings, each at most u
relative to |s| + |bias| -- and once to the output type (eps / 2; below the fp16 normal range half of 2^-24 absolute)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import gazenerf_amd as G
from gazenerf_amd import _lib, _torch_ext, int8

DEV = "cuda"
gpu = pytest.mark.gpu
TYPES = (torch.float32, torch.bfloat16, torch.float16)


# ---- the plain implementation, in 64 bits on the CPU -----------------------------------------------------------------------------
def ref_rows(x):
    """x [..., K] -> (q float64 whole steps, scale float32)."""
    x = x.detach().cpu().double()
    a = x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    a = torch.where(bad, torch.ones_like(a), a)
    per = (127 / a).float().double()
    q = torch.where(bad, torch.zeros_like(x), torch.round((torch.where(bad, torch.zeros_like(x), x) * per).float().double()))
    s = torch.where(bad, torch.full_like(a, math.nan), a / 127).float().squeeze(-1)
    return q, s


def ref_linear(q, s, wq, ws, bias, leaky):
    """(y, bound on the fp32 epilogue's error), rows last-axis."""
    q, s, wq, ws = q.cpu().double(), s.cpu().double(), wq.cpu().double(), ws.cpu().double()
    t = (q @ wq.t()) * s.unsqueeze(-1) * ws
    b = bias.cpu().double() if bias is not None else torch.zeros(wq.shape[0], dtype=torch.float64)
    y = t + b
    if leaky:
        y = torch.where(y > 0, y, y * 0.2)
    return y, 6 * 2.0 ** -24 * (t.abs() + b.abs())


def assert_linear(y, ref, bound):
    y = y.detach().cpu()
    tiny = 2.0 ** -25 if y.dtype == torch.float16 else 2.0 ** -149
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(y), nan)
    big = torch.finfo(y.dtype).max
    d = (y.double() - ref).abs()
    lim = bound + torch.finfo(y.dtype).eps / 2 * (ref.abs() + bound) + tiny
    ok = (d <= lim) | nan | ((ref.abs() + bound >= big * (1 - 2.0 ** -12)) & (y.double().sign() == ref.sign()))
    assert bool(ok.all()), (int((~ok).sum()), float((d - lim)[~ok].max()))


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def features(shape, axis, seed, dtype=torch.float32):
    """Maps with channels of different size, zero pixels, and a few rows of extreme size."""
    g = gen(seed)
    x = torch.randn(shape, generator=g)
    v = [1] * len(shape)
    v[axis] = shape[axis]
    x = x * torch.exp(torch.randn(shape[axis], generator=g)).view(v)
    v = list(shape)
    v[axis] = 1
    return (x * (torch.rand(v, generator=g) > 0.1)).to(dtype)


def weights(o, k, seed):
    w = torch.randn(o, k, generator=gen(seed)) * math.sqrt(2.0 / (o + k))
    return w, torch.randn(o, generator=gen(seed + 1)) * 0.1


def new_cache(n, p, c, seed=0):
    """A cache whose every byte (the ones between the rows too) holds a known pattern."""
    store = torch.randint(-128, 128, (n, p, int8.row_pitch(c)), generator=gen(seed), dtype=torch.int8).to(DEV)
    return store, store[..., :c], torch.rand(n, p, generator=gen(seed + 1)).to(DEV)


def linear_ref_of(x, w_q, w_s, bias, leaky):
    q, s = ref_rows(x)
    return ref_linear(q, s, w_q, w_s, bias, leaky)


# ---- CPU: refusals ---------------------------------------------------------------------------------------------------------------
def cpu_args():
    w = torch.zeros(5, 16, dtype=torch.int8)
    return dict(x=torch.zeros(3, 16), w_q=w, w_scale=torch.ones(5), bias=torch.zeros(5))


@pytest.mark.parametrize("change, error, match", [
    (dict(x=torch.zeros(3, 17)), ValueError, "channels"),
    (dict(x=torch.zeros(3, 16, dtype=torch.float64)), TypeError, "float32"),
    (dict(x=[1.0]), TypeError, "tensor"),
    (dict(w_q=torch.zeros(5, 16)), TypeError, "int8"),
    (dict(w_q=torch.zeros(5, 4, 4, dtype=torch.int8)), ValueError, "dimensions"),
    (dict(w_q=torch.zeros(0, 16, dtype=torch.int8), w_scale=torch.ones(0), bias=None), ValueError, "empty"),
    (dict(w_scale=torch.ones(4)), ValueError, "w_scale"),
    (dict(w_scale=torch.ones(5, dtype=torch.float64)), TypeError, "w_scale"),
    (dict(bias=torch.zeros(6)), ValueError, "bias"),
    (dict(bias=torch.zeros(5, dtype=torch.bfloat16)), TypeError, "bias"),
    (dict(x_scale=torch.ones(3)), ValueError, "quantised by the call"),
    (dict(slots=torch.zeros(1, dtype=torch.int64)), ValueError, "quantised by the call"),
    (dict(channels_first=True), ValueError, r"\[B, K"),
    (dict(out_dtype=torch.float64), TypeError, "out_dtype"),
    (dict(out_dtype=torch.int8), TypeError, "out_dtype"),
    (dict(x=torch.zeros(3, 16, dtype=torch.int8)), ValueError, "x_scale"),
    (dict(x=torch.zeros(3, 16, dtype=torch.int8), x_scale=torch.ones(4)), ValueError, "x_scale"),
    (dict(x=torch.zeros(3, 16, dtype=torch.int8), x_scale=torch.ones(3, dtype=torch.float16)), TypeError, "x_scale"),
    (dict(x=torch.zeros(3, 16, dtype=torch.int8), x_scale=torch.ones(3), channels_first=True), ValueError, r"\[n, P, K\]"),
    (dict(x=torch.zeros(3, 16, dtype=torch.int8), x_scale=torch.ones(3), slots=torch.zeros(1, dtype=torch.int64)), ValueError, r"\[n, P, K\]"),
    (dict(x=torch.zeros(2, 3, 16, dtype=torch.int8), x_scale=torch.ones(2, 3), slots=torch.zeros(1, dtype=torch.int32)), TypeError, "int64"),
    (dict(x=torch.zeros(0, 3, 16, dtype=torch.int8), x_scale=torch.ones(0, 3), slots=torch.zeros(1, dtype=torch.int64)), ValueError, "empty"),
    (dict(x=torch.zeros(1, 131072), w_q=torch.zeros(1, 131072, dtype=torch.int8), w_scale=torch.ones(1), bias=None), ValueError, "131071"),
    (dict(), RuntimeError, "CUDA/ROCm"),
])
@pytest.mark.parametrize("binding", ["auto", "ctypes"])
def test_linear_refusals(change, error, match, binding, monkeypatch, lib_built):
    monkeypatch.setenv("GNR_BINDING", binding)
    a = cpu_args()
    a.update(change)
    with pytest.raises(error, match=match):
        G.int8_linear(a.pop("x"), a.pop("w_q"), a.pop("w_scale"), a.pop("bias"), **a)


@pytest.mark.parametrize("binding", ["auto", "ctypes"])
def test_cache_refusals(binding, monkeypatch, lib_built):
    monkeypatch.setenv("GNR_BINDING", binding)
    q, s, slots, maps = torch.zeros(4, 6, 16, dtype=torch.int8), torch.zeros(4, 6), torch.zeros(2, dtype=torch.int64), torch.zeros(2, 16, 6)
    cases = [((q.float(), s, slots, maps), TypeError, "q must be int8"), ((q[0], s, slots, maps), ValueError, "dimensions"),
             ((q, s[:, :5], slots, maps), ValueError, "scale must have shape"), ((q, s.double(), slots, maps), TypeError, "scale"),
             ((q, s, slots.int(), maps), TypeError, "slots"), ((q, s, slots[None], maps), ValueError, "dimensions"),
             ((q, s, slots, maps[:1]), ValueError, "maps must be"), ((q, s, slots, maps[:, :15]), ValueError, "maps must be"),
             ((q, s, slots, maps[:, :, :5]), ValueError, "maps must be"), ((q, s, slots, maps.double()), TypeError, "maps"),
             ((q.transpose(1, 2).contiguous().transpose(1, 2), s, slots, maps), ValueError, "strides"),
             ((q[:1].expand(4, 6, 16), s, slots, maps), ValueError, "strides"), ((q, s[:1].expand(4, 6), slots, maps), ValueError, "strides"),
             ((q[:0], s[:0], slots, maps), ValueError, "empty"), ((q, s, slots, maps), RuntimeError, "CUDA/ROCm")]
    for args, error, match in cases:
        with pytest.raises(error, match=match):
            G.write_featmaps(*args)
        if args[3] is maps:
            with pytest.raises(error, match=match):
                G.read_featmaps(*args[:3])
    with pytest.raises(TypeError, match="out_dtype"):
        G.read_featmaps(q, s, slots, torch.int8)
    for bad, error in ((torch.zeros(3, dtype=torch.int8), TypeError), (torch.zeros(3, 0), ValueError), (torch.zeros(()), ValueError), (None, TypeError)):
        with pytest.raises(error):
            G.quantize_rows(bad)
    with pytest.raises(ValueError, match=r"\[B, K"):
        G.quantize_rows(torch.zeros(3, 4), channels_first=True)
    for n in ((0, 4, 4), (4, 0, 4), (4, 4, 0)):
        with pytest.raises(ValueError, match=">= 1"):
            G.FeatureMapCache(*n, device="cpu")
    with pytest.raises(IndexError, match="slot 4"):
        G.FeatureMapCache(4, 3, 2, device="cpu").slots([0, 4])


def test_no_backward(lib_built):
    """Inference only: a call that would need a gradient is refused before anything runs."""
    x, w = torch.zeros(3, 16, requires_grad=True), torch.zeros(5, 16, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="no backward"):
        G.int8_linear(x, w, torch.ones(5))
    with pytest.raises(RuntimeError, match="no backward"):
        G.int8_linear(x.detach(), w, torch.ones(5), torch.zeros(5, requires_grad=True))
    with pytest.raises(RuntimeError, match="no backward"):
        G.quantize_rows(x)
    with pytest.raises(RuntimeError, match="no backward"):
        G.write_featmaps(torch.zeros(1, 3, 16, dtype=torch.int8), torch.zeros(1, 3), torch.zeros(1, dtype=torch.int64), x.t()[None])
    cache = torch.zeros(1, 3, 16, dtype=torch.int8), torch.ones(1, 3, requires_grad=True), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no backward"):
        G.write_featmaps(*cache, torch.zeros(1, 16, 3))
    with pytest.raises(RuntimeError, match="no backward"):
        G.read_featmaps(*cache)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA/ROCm"):       # no gradient wanted: the next check speaks
        G.int8_linear(x, w, torch.ones(5))


def test_no_forward_mode_gradient_and_no_trace(lib_built):
    """A tangent would be dropped (``requires_grad`` is False on a dual tensor), a trace would hold the result as a constant: both are refused."""
    from torch.autograd import forward_ad
    w, ones, slots = torch.zeros(5, 16, dtype=torch.int8), torch.ones(5), torch.zeros(1, dtype=torch.int64)
    q, s = torch.zeros(1, 3, 16, dtype=torch.int8), torch.ones(1, 3)
    params = {n: torch.zeros(1) for n in ("a", "b")}
    calls = [lambda d: G.quantize_rows(d(torch.zeros(3, 16))), lambda d: G.int8_linear(d(torch.zeros(3, 16)), w, ones),
             lambda d: G.int8_linear(torch.zeros(3, 16), w, d(ones)), lambda d: G.int8_linear(torch.zeros(3, 16), w, ones, d(torch.zeros(5))),
             lambda d: G.int8_linear(q[0], w, ones, x_scale=d(s[0])), lambda d: G.write_featmaps(q, s, slots, d(torch.zeros(1, 16, 3))),
             lambda d: G.write_featmaps(q, d(s), slots, torch.zeros(1, 16, 3)), lambda d: G.read_featmaps(q, d(s), slots),
             lambda d: G.neural_render_int8(d(torch.zeros(1, 4, 16, 16)), params), lambda d: G.neural_render_int8(torch.zeros(1, 4, 16, 16), dict(params, b=d(ones)))]
    for call in calls:
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), forward_ad.dual_level():
                with pytest.raises(RuntimeError, match="no forward-mode gradient"):
                    call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
    with torch.no_grad(), pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda t: G.quantize_rows(t).scale, torch.zeros(3, 16), check_trace=False)


def test_c_entries_refuse(lib_built):
    """The C ABI checks every size it indexes with before it launches anything (bogus pointers: nothing may be dereferenced)."""
    lib = _lib.load()

    def rows(**kw):
        p = _lib.GnrRowsProblem()
        p.dtype, p.channels_first, p.batch, p.n_pix, p.channels = 0, 1, 2, 8, 5
        p.x = p.q = p.scale = p.slots = 4096
        p.x_batch, p.x_stride, p.q_batch, p.q_pitch, p.scale_batch, p.n_slots = 40, 8, 128, 16, 8, 3
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    for fn in (lib.gnr_quantize_rows, lib.gnr_read_rows):
        assert fn(None, None) != 0
        for kw, word in ((dict(struct_size=8), "struct_size"), (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(batch=-1), "batch"),
                         (dict(n_pix=-1), "n_pix"), (dict(channels=0), "channels"), (dict(x=None), "NULL"), (dict(q=None), "NULL"),
                         (dict(scale=None), "NULL"), (dict(x_stride=-1), "stride"), (dict(q_pitch=4), "q_pitch"), (dict(n_slots=0), "n_slots"),
                         (dict(n_pix=1 << 31), "2^31"), (dict(channels_first=0), "channels-first")):
            assert fn(C.byref(rows(**kw)), None) != 0, kw
            assert word in lib.gnr_last_error().decode(), (kw, lib.gnr_last_error())
        huge = dict(dtype=1, batch=1, n_pix=1 << 31, channels=4096, q_pitch=4096, slots=None, n_slots=0)      # more threads than a grid counts
        assert fn(C.byref(rows(**huge)), None) != 0 and "exceed one launch" in lib.gnr_last_error().decode()
        assert fn(C.byref(rows(batch=0)), None) == 0 and fn(C.byref(rows(n_pix=0)), None) == 0      # an empty call

    def lin(**kw):
        p = _lib.GnrInt8Problem()
        p.x_type, p.y_type, p.batch, p.k, p.o, p.n_pix = 3, 0, 2, 20, 5, 8
        p.x = p.x_scale = p.slots = p.w = p.w_scale = p.bias = p.y = 4096
        p.x_batch, p.x_stride, p.x_scale_batch, p.n_slots, p.w_pitch = 256, 32, 8, 3, 32
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    bad = ((dict(struct_size=8), "struct_size"), (dict(x_type=4), "x_type"), (dict(y_type=3), "y_type"), (dict(batch=-1), "batch"), (dict(k=0), "k and o"),
           (dict(o=0), "k and o"), (dict(k=131072, w_pitch=131072), "exceeds"), (dict(o=(1 << 27) + 1), "exceeds"), (dict(x_channels_first=1), "channels last"),
           (dict(x_type=0), "slots"), (dict(n_slots=0), "n_slots"), (dict(n_pix=1 << 31), "2^31"), (dict(x=None), "NULL"), (dict(w=None), "NULL"),
           (dict(y=None), "NULL"), (dict(w_scale=None), "NULL"), (dict(x_scale=None), "x_scale"), (dict(w=4097), "16-byte"), (dict(w_pitch=24), "16-byte"),
           (dict(w_pitch=16), "16-byte"), (dict(x=4100), "16-byte"), (dict(x_stride=40), "16-byte"), (dict(x_stride=16), "16-byte"),
           (dict(x_batch=8), "16-byte"), (dict(x_scale_batch=-1), "negative"))
    for kw, word in bad:
        assert lib.gnr_int8_linear(C.byref(lin(**kw)), None, 0, None) != 0, kw
        assert word in lib.gnr_last_error().decode(), (kw, lib.gnr_last_error())
        assert lib.gnr_int8_linear_workspace_bytes(C.byref(lin(**kw))) == 0, kw
    assert lib.gnr_int8_linear(None, None, 0, None) != 0
    assert lib.gnr_int8_linear(C.byref(lin(batch=0)), None, 0, None) == 0
    assert lib.gnr_int8_linear(C.byref(lin(batch=1 << 25, n_pix=33, y_channels_first=1)), None, 0, None) != 0
    assert "exceed one launch" in lib.gnr_last_error().decode()
    flt = dict(x_type=0, slots=None, n_slots=0)
    need = lib.gnr_int8_linear_workspace_bytes(C.byref(lin(**flt)))
    assert need >= 16 * 32 + 16 * 4                                     # the rows on their pitch and their scales
    assert lib.gnr_int8_linear(C.byref(lin(**flt)), 4096, need - 256, None) != 0 and "workspace" in lib.gnr_last_error().decode()
    assert lib.gnr_int8_linear(C.byref(lin(**flt)), 4100, need, None) != 0 and "256-byte" in lib.gnr_last_error().decode()


def test_plain_rows_definition():
    """The reference of this file itself: zero rows, rows below the floor, rows with Inf / NaN, steps on a border (ties to even)."""
    x = torch.tensor([[0.0, 0.0], [127.0, 0.5], [127.0, 1.5], [127.0, -2.5], [1.0, -3.0], [2.0 ** -120, 0.0], [math.inf, 1.0], [math.nan, 1.0]])
    q, s = ref_rows(x)
    assert q.tolist()[:5] == [[0, 0], [127, 0], [127, 2], [127, -2], [42, -127]] and q[5].tolist() == [0, 0] and q[6:].abs().max() == 0
    assert s[0] == s[5] == torch.tensor(2.0 ** -100 / 127) and s[1] == 1.0 and bool(torch.isnan(s[6:]).all())


# ---- GPU: rows -------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, k", [(1, 1), (1, 7), (3, 16), (65, 17), (33, 64), (17, 129), (5, 258), (9, 517), (4, 1030), (3, 2048), (2, 4099), (3, 9001)])
def test_quantize_rows(dtype, n, k):
    x = features((n, k), 1, 10 * n + k, dtype)
    x.view(-1)[0] = 3.0
    r = G.quantize_rows(x.to(DEV))
    q, s = ref_rows(x)
    assert r.q.dtype == torch.int8 and r.q.shape == (n, k) and (n == 1 or r.q.stride(0) == int8.row_pitch(k))
    assert torch.equal(r.q.cpu().double(), q) and torch.equal(r.scale.cpu(), s)


@gpu
def test_quantize_rows_special_values():
    """Zero rows, rows below the floor, the largest values, denormals, and Inf / NaN in one place of a row."""
    for k in (1, 3, 64, 300, 3000):
        x = torch.randn(11, k, generator=gen(k))
        x[0] = 0
        x[1] = x[1] * 2.0 ** -130
        x[2] = x[2] * 2.0 ** -101
        x[3] = torch.finfo(torch.float32).max
        x[4, k // 2], x[5, k - 1], x[6, 0] = math.inf, -math.inf, math.nan
        x[7] = -0.0
        x[8] = 2.0 ** -149
        x[9, 0] = 127.0
        x[9, 1:] = torch.arange(1, k) % 100 + 0.5                          # every value on a border between two steps
        r = G.quantize_rows(x.to(DEV))
        q, s = ref_rows(x)
        assert torch.equal(r.q.cpu().double(), q)
        assert torch.equal(torch.isnan(r.scale.cpu()), torch.isnan(s)) and torch.equal(r.scale.cpu().nan_to_num(), s.nan_to_num())
        m = G.quantize_rows(x.t()[None].contiguous().to(DEV), channels_first=True)      # the other layout's kernel, same rows
        assert torch.equal(m.q[0].cpu(), r.q.cpu()) and torch.equal(m.scale[0].cpu().nan_to_num(), s.nan_to_num())


@gpu
def test_quantize_rows_shapes_and_strides():
    x = features((4, 6, 5, 40), 3, 3)
    xd = x.to(DEV)
    q, s = ref_rows(x)
    r = G.quantize_rows(xd)
    assert r.q.shape == x.shape and r.scale.shape == x.shape[:-1] and torch.equal(r.q.cpu().double(), q) and torch.equal(r.scale.cpu(), s)
    one = G.quantize_rows(xd[0, 0, 0])
    assert one.q.shape == (40,) and one.scale.shape == () and torch.equal(one.q.cpu().double(), q[0, 0, 0])
    for view in (xd[:, ::2], xd[..., 3:38], xd[:, :, 1], xd.transpose(0, 1), xd[..., ::3], xd[1:2].expand(3, 6, 5, 40), xd[0].transpose(0, 2)):
        q, s = ref_rows(view)
        r = G.quantize_rows(view)
        assert torch.equal(r.q.cpu().double(), q) and torch.equal(r.scale.cpu(), s)
    for view in (xd[:, :, 0], xd[0].transpose(1, 2), xd.permute(0, 3, 1, 2), xd[0:1].expand(3, 6, 5, 40)[:, :, 1], xd[..., 3:38]):
        r = G.quantize_rows(view, channels_first=True)
        q, s = ref_rows(view.flatten(2).transpose(1, 2))
        assert torch.equal(r.q.cpu().double(), q) and torch.equal(r.scale.cpu(), s)
    for shape in ((0, 8), (3, 0, 8), (0,) + (2, 8)):
        r = G.quantize_rows(torch.empty(shape, device=DEV))
        assert r.q.shape == shape and r.scale.shape == shape[:-1]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b, c, p", [(1, 1, 1), (2, 3, 5), (1, 64, 33), (3, 129, 64), (2, 258, 100), (1, 515, 37), (1, 1024, 65), (1, 2047, 40), (1, 2300, 34), (1, 4500, 9)])
def test_maps_to_rows(dtype, b, c, p):
    x = features((b, c, p), 1, b + c + p, dtype)
    r = G.quantize_rows(x.to(DEV), channels_first=True)
    q, s = ref_rows(x.transpose(1, 2))
    assert torch.equal(r.q.cpu().double(), q) and torch.equal(r.scale.cpu(), s)


# ---- GPU: the cache --------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c, p", [(1, 1), (16, 64), (129, 37), (258, 256), (1024, 65), (2500, 33)])
def test_cache_write_and_read(dtype, c, p):
    n = 7
    store, q, scale = new_cache(n, p, c)
    before, sbefore = store.cpu(), scale.cpu()
    maps = features((3, c, p), 1, c, dtype)
    slots = torch.tensor([5, 0, 2], device=DEV)
    G.write_featmaps(q, scale, slots, maps.to(DEV))
    want_q, want_s = ref_rows(maps.transpose(1, 2))
    expect, sexpect = before.clone(), sbefore.clone()
    expect[[5, 0, 2], :, :c] = want_q.to(torch.int8)                       # nothing else moves: other slots, bytes behind the rows
    sexpect[[5, 0, 2]] = want_s
    assert torch.equal(store.cpu(), expect) and torch.equal(scale.cpu(), sexpect)
    order = torch.tensor([2, 6, 5, 5, 0], device=DEV)
    for out in TYPES:
        got = G.read_featmaps(q, scale, order, out)
        want = (expect[order.cpu(), :, :c].float() * sexpect[order.cpu()].unsqueeze(-1)).transpose(1, 2).to(out)
        assert got.shape == (5, c, p) and torch.equal(got.cpu(), want)


@gpu
def test_cache_slots_outside_and_repeated():
    c, p, n = 70, 50, 4
    store, q, scale = new_cache(n, p, c)
    before, sbefore = store.cpu(), scale.cpu()
    maps = features((6, c, p), 1, 1).to(DEV)
    G.write_featmaps(q, scale, torch.tensor([1, -1, 1, n, 3, 1], device=DEV), maps)      # slot 1 three times: the last stays
    want_q, want_s = ref_rows(maps.transpose(1, 2))
    expect, sexpect = before.clone(), sbefore.clone()
    expect[[1, 3], :, :c], sexpect[[1, 3]] = want_q[[5, 4]].to(torch.int8), want_s[[5, 4]]
    assert torch.equal(store.cpu(), expect) and torch.equal(scale.cpu(), sexpect)
    far = torch.tensor([3, -1, n, 2 ** 40, -2 ** 40, 1], device=DEV)
    got = G.read_featmaps(q, scale, far).cpu()
    assert torch.equal(got[0], (want_q[4].float() * want_s[4].unsqueeze(-1)).t()) and torch.equal(got[5], (want_q[5].float() * want_s[5].unsqueeze(-1)).t())
    assert bool((got[[1, 4]] == 0).all()) and bool(torch.isnan(got[[2, 3]]).all())
    w, b = weights(33, c, 5)
    wq = G.quantize_rows(w.to(DEV))
    for cf in (False, True):
        y = G.int8_linear(q, wq.q, wq.scale, b.to(DEV), x_scale=scale, slots=far, channels_first=cf).cpu()
        y = y.transpose(1, 2) if cf else y
        assert torch.equal(y[1], b.expand(p, 33)) and torch.equal(y[4], y[1]) and bool(torch.isnan(y[[2, 3]]).all())
        ref, bound = ref_linear(want_q[4], want_s[4], wq.q, wq.scale, b, False)
        assert_linear(y[0], ref, bound)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    G.write_featmaps(q, scale, none, maps[:0])
    assert G.read_featmaps(q, scale, none).shape == (0, c, p)
    assert G.int8_linear(q, wq.q, wq.scale, x_scale=scale, slots=none).shape == (0, p, 33)
    assert torch.equal(store.cpu(), expect)


@gpu
def test_cache_strides():
    """A cache that is a view (every second slot, some of the channels) and maps that are views."""
    big = torch.zeros(8, 30, 96, dtype=torch.int8, device=DEV)
    q, scale = big[1::2, 2:22, 16:57], torch.zeros(4, 64, device=DEV)[:, 5:25]
    maps = features((3, 60, 4, 5), 1, 9).to(DEV)[:, 7:48].permute(0, 1, 3, 2)
    slots = torch.tensor([9, 0, 9, 3, 9, 1], device=DEV)[1::2]
    G.write_featmaps(q, scale, slots, maps)
    want_q, want_s = ref_rows(maps.flatten(2).transpose(1, 2))
    mark = torch.zeros(8, 30, 96, dtype=torch.int8)
    mark[1::2, 2:22, 16:57][[0, 3, 1]] = want_q.to(torch.int8)
    assert torch.equal(big.cpu(), mark) and torch.equal(scale.cpu()[[0, 3, 1]], want_s)
    got = G.read_featmaps(q, scale, slots)
    assert torch.equal(got.cpu(), (want_q.float() * want_s.unsqueeze(-1)).transpose(1, 2))
    w, b = weights(20, 41, 3)
    wq = G.quantize_rows(w.to(DEV))
    ref, bound = ref_linear(want_q, want_s, wq.q, wq.scale, b, True)
    assert_linear(G.int8_linear(q, wq.q, wq.scale, b.to(DEV), x_scale=scale, slots=slots, leaky=True), ref, bound)


@gpu
def test_quantize_more_rows_than_one_launch():
    """A grid counts its threads in 32 bits: 16 lanes a row reach that at 2^28 rows, launches end at 2^27."""
    n, at = (1 << 28) + 33, 1 << 27
    x = torch.full((n, 1), 1.5, dtype=torch.bfloat16, device=DEV)
    probe = torch.tensor([0, 1, at - 1, at, at + 1, 2 * at - 1, 2 * at, n - 2, n - 1], device=DEV)
    x[probe] = torch.tensor([[-1.0], [0.0], [2.5], [-3.25], [1e-20], [-7.0], [0.5], [1e20], [-0.125]], dtype=torch.bfloat16, device=DEV)
    q, scale = G.quantize_rows(x)
    want_q, want_s = ref_rows(x[probe])
    assert torch.equal(q[probe].cpu().double(), want_q) and torch.equal(scale[probe].cpu(), want_s)
    rest = torch.ones(n, dtype=torch.bool, device=DEV)
    rest[probe] = False
    assert bool((scale[rest] == ref_rows(torch.tensor([1.5]))[1].item()).all()) and bool((q[:, 0][rest] == 127).all())


@gpu
def test_cache_offsets_beyond_32_bits():
    """Slots whose bytes lie behind 2^32."""
    c, p, n = 1024, 4096, 1100
    q, scale = int8.empty_rows(n, p, c, device=DEV), torch.zeros(n, p, device=DEV)
    maps = features((2, c, p), 1, 2, torch.bfloat16).to(DEV)
    slots = torch.tensor([n - 1, 1025], device=DEV)
    assert (n - 1) * p * c > 2 ** 32
    G.write_featmaps(q, scale, slots, maps)
    want_q, want_s = ref_rows(maps.transpose(1, 2))
    assert torch.equal(q[slots].cpu().double(), want_q) and torch.equal(scale[slots].cpu(), want_s)
    got = G.read_featmaps(q, scale, slots)
    assert torch.equal(got.cpu(), (want_q.float() * want_s.unsqueeze(-1)).transpose(1, 2))
    w, _ = weights(40, c, 3)
    wq = G.quantize_rows(w.to(DEV))
    ref, bound = ref_linear(want_q, want_s, wq.q, wq.scale, None, False)
    assert_linear(G.int8_linear(q, wq.q, wq.scale, x_scale=scale, slots=slots), ref, bound)


@gpu
def test_feature_map_cache():
    cache = G.FeatureMapCache(5, 30, 24, device=DEV)
    maps = features((2, 30, 4, 6), 1, 4).to(DEV)
    cache.write([3, 1], maps)
    assert bool(torch.isnan(cache.read(0)).all()) and cache.n_slots == 5                    # never written
    want_q, want_s = ref_rows(maps.flatten(2).transpose(1, 2))
    want = (want_q.float() * want_s.unsqueeze(-1)).transpose(1, 2)
    assert torch.equal(cache.read((1, 3)).cpu(), want[[1, 0]]) and torch.equal(cache.read(torch.tensor([3], device=DEV), torch.bfloat16).cpu(), want[:1].bfloat16())
    # half a step of the row's scale, plus the rounding of the value to fp32
    err = (cache.read([3, 1]).cpu().double() - maps.flatten(2).cpu().double()).abs()
    step = want_s.double().unsqueeze(1)
    assert bool((err <= step * (0.5 + 127 * 2.0 ** -22)).all())
    assert torch.equal(cache.read(np.int64(3)), cache.read([np.int32(3)]))
    w, b = weights(17, 30, 1)
    wq = G.quantize_rows(w.to(DEV))
    ref, bound = ref_linear(want_q, want_s, wq.q, wq.scale, b, True)
    y = cache.linear([3, 1], wq.q, wq.scale, b.to(DEV), leaky=True, channels_first=True)
    assert_linear(y.transpose(1, 2), ref, bound)


# ---- GPU: the product ------------------------------------------------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 16, 5), (1, 300, 700), (2, 517, 259), (3, 64, 32), (5, 2048, 96), (15, 129, 33), (16, 258, 516), (17, 63, 65), (31, 1000, 40),
         (33, 65, 130), (64, 32, 64), (65, 31, 129), (130, 258, 260), (200, 516, 97), (257, 96, 200), (300, 1040, 31), (513, 17, 513), (700, 129, 64),
         (1025, 48, 16), (2000, 64, 32)]


@gpu
@pytest.mark.parametrize("n, k, o", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_rows(n, k, o, dtype):
    x = features((n, k), 1, n + k + o, dtype)
    w, b = weights(o, k, o)
    wq = G.quantize_rows(w.to(DEV))
    for leaky, bias, out in ((True, b, dtype), (False, None, torch.float32)):
        ref, bound = linear_ref_of(x, wq.q, wq.scale, bias, leaky)
        y = G.int8_linear(x.to(DEV), wq.q, wq.scale, None if bias is None else bias.to(DEV), leaky=leaky, out_dtype=out)
        assert y.dtype == out and y.shape == (n, o)
        assert_linear(y, ref, bound)


@gpu
@pytest.mark.parametrize("b, k, o, p", [(1, 5, 3, 1), (2, 64, 32, 50), (1, 129, 64, 130), (3, 258, 516, 100), (2, 40, 33, 257), (1, 516, 100, 600), (2, 64, 31, 300), (4, 32, 129, 7)])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_maps(b, k, o, p, dtype):
    x = features((b, k, p), 1, b + k + o + p, dtype)
    w, bias = weights(o, k, o)
    wq = G.quantize_rows(w.to(DEV))
    ref, bound = linear_ref_of(x.transpose(1, 2), wq.q, wq.scale, bias, True)
    for out in (dtype, torch.float32):
        y = G.int8_linear(x.to(DEV), wq.q, wq.scale, bias.to(DEV), leaky=True, channels_first=True, out_dtype=out)
        assert y.dtype == out and y.shape == (b, o, p)
        assert_linear(y.transpose(1, 2), ref, bound)
    q = G.quantize_rows(x.to(DEV), channels_first=True)                       # the same rows, quantised before
    again = G.int8_linear(q.q, wq.q, wq.scale, bias.to(DEV), x_scale=q.scale, leaky=True, channels_first=True, out_dtype=torch.float32)
    assert torch.equal(again, y)                                            # the sum is exact, the epilogue the same: equal bits
    rows = G.int8_linear(q.q, wq.q, wq.scale, bias.to(DEV), x_scale=q.scale, leaky=True, out_dtype=torch.float32)
    assert_linear(rows, ref, bound)


@gpu
@pytest.mark.parametrize("n, k, o", [
    (150, 1430, 250), (100, 2050, 834), (30, 100, 9000), (64, 40, 5000),         # blocks of 16, 32 and 64 rows whose waves share K
    (1030, 129, 259), (9000, 48, 31), (5000, 130, 63),                           # 64 x 64 tiles, layers of at most 32 and 64 outputs
    (4100, 70, 1030), (6500, 517, 2050), (4090, 515, 4090)])                     # 128 x 128, 128 x 256, 256 x 256 tiles
def test_linear_every_tile(n, k, o):
    """8-bit rows with bytes behind their channels, as rows and as two maps, every type of result; the sums in 64 bits (whole numbers: exact)."""
    g = gen(n + k + o)
    x = torch.randint(-128, 128, (n, int8.row_pitch(k, 16)), generator=g, dtype=torch.int8).to(DEV)[:, :k]
    w = torch.randint(-128, 128, (o, int8.row_pitch(k, 16)), generator=g, dtype=torch.int8).to(DEV)[:, :k]
    xs, ws, b = torch.rand(n, generator=g) * 0.02, torch.rand(o, generator=g) * 0.02, torch.randn(o, generator=g)
    xs[n // 2], xs[n - 1] = 0.0, math.nan
    t = (x.double() @ w.double().t()).cpu() * xs.double()[:, None] * ws.double()
    y = t + b.double()
    ref, bound = torch.where(y < 0, y * 0.2, y), 6 * 2.0 ** -24 * (t.abs() + b.double().abs())
    args = w, ws.to(DEV), b.to(DEV)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        assert_linear(G.int8_linear(x, *args, x_scale=xs.to(DEV), leaky=True, out_dtype=out), ref, bound)
        maps = G.int8_linear(x.view(2, n // 2, k), *args, x_scale=xs.to(DEV).view(2, -1), leaky=True, channels_first=True, out_dtype=out)
        assert_linear(maps.transpose(1, 2).reshape(n, o), ref, bound)


@gpu
def test_linear_any_bytes():
    """8-bit rows a caller made (the value -128, bytes behind the channels that are not zero), sums that need more than 24 bits."""
    for n, k, o in ((5, 130000, 3), (300, 2050, 70), (1, 999, 40)):
        g = gen(k)
        store_x = torch.full((n, int8.row_pitch(k) + 32), -77, dtype=torch.int8)
        store_w = torch.full((o, int8.row_pitch(k) + 16), 55, dtype=torch.int8)
        store_x[:, :k] = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
        store_w[:, :k] = torch.randint(-128, 128, (o, k), generator=g, dtype=torch.int8)
        store_x[0, :k] = -128
        store_w[0, :k] = -128                                                # 128 * 128 * k: the largest sum there is
        xs, ws = torch.rand(n, generator=g), torch.rand(o, generator=g)
        ref, bound = ref_linear(store_x[:, :k], xs, store_w[:, :k], ws, None, False)
        dx, dw = store_x.to(DEV)[:, :k], store_w.to(DEV)[:, :k]
        assert_linear(G.int8_linear(dx, dw, ws.to(DEV), x_scale=xs.to(DEV)), ref, bound)
        # the same values where the product cannot read them in place: odd pitch, odd start
        odd_x = torch.zeros(n, k + 3, dtype=torch.int8, device=DEV)[:, 3:]
        odd_x.copy_(dx)
        odd_w = torch.zeros(o * k + 1, dtype=torch.int8, device=DEV)[1:].view(o, k)
        odd_w.copy_(dw)
        assert_linear(G.int8_linear(odd_x, odd_w, ws.to(DEV), x_scale=xs.to(DEV)), ref, bound)


@gpu
def test_linear_shapes_strides_and_empties():
    w, b = weights(24, 40, 2)
    wq = G.quantize_rows(w.to(DEV))
    x = features((3, 4, 5, 40), 3, 8)
    xd = x.to(DEV)
    bd = b.to(DEV)
    for view in (xd, xd[0, 0, 0], xd[:, ::2], xd.transpose(0, 2), xd[1:2].expand(5, 4, 5, 40), xd[:, :, 1]):
        ref, bound = linear_ref_of(view, wq.q, wq.scale, b, False)
        y = G.int8_linear(view, wq.q, wq.scale, bd)
        assert y.shape == view.shape[:-1] + (24,)
        assert_linear(y, ref, bound)
    m = xd.permute(0, 3, 1, 2)                                               # [3, 40, 4, 5], channels last in memory
    y = G.int8_linear(m, wq.q, wq.scale, bd, channels_first=True)
    ref, bound = linear_ref_of(xd.reshape(3, 20, 40), wq.q, wq.scale, b, False)
    assert y.shape == (3, 24, 4, 5)
    assert_linear(y.flatten(2).transpose(1, 2), ref, bound)
    big = torch.zeros(48, 64, device=DEV)                                    # strided scale and bias
    big[::2, 3], big[1::2, 3] = wq.scale, bd
    assert torch.equal(G.int8_linear(xd, wq.q, big[::2, 3], big[1::2, 3]), G.int8_linear(xd, wq.q, wq.scale, bd))
    assert G.int8_linear(torch.empty(0, 40, device=DEV), wq.q, wq.scale).shape == (0, 24)
    assert G.int8_linear(torch.empty(2, 40, 0, device=DEV), wq.q, wq.scale, channels_first=True).shape == (2, 24, 0)
    with pytest.raises(RuntimeError, match="one device|must live on"):
        G.int8_linear(xd, wq.q.cpu(), wq.scale)


def test_rows_of_three_dimensions_are_one_entry():
    """The ctypes binding's view of floating rows [b, n, K]: one entry where they stand one behind the other, the same values always."""
    x = torch.arange(4 * 6 * 5.0).reshape(4, 6, 5)
    for t, one in ((x, True), (x[:, :1], True), (x[:1], False), (x[:, :5], False), (x[:, ::2], True), (x[::2], False), (x[:, :0], False), (x[:, 2:3].expand(4, 3, 5), False)):
        y = int8._one_entry(t)
        assert torch.equal(y.reshape(-1, 5), t.reshape(-1, 5)) and (y.shape[0] == 1 and t.shape[0] > 1) == one, t.shape


@gpu
@pytest.mark.parametrize("binding", ["auto", "ctypes"])
@pytest.mark.parametrize("k", [40, 517])
def test_linear_rows_of_three_dimensions(k, binding, monkeypatch):
    """The same bits however the rows are counted, and no workspace for [4, 4, K] where [16, K] needs none."""
    if binding == "ctypes":
        monkeypatch.setattr(_torch_ext, "active", lambda: None)
    w, b = weights(33, k, 3)
    wq, bd = G.quantize_rows(w.to(DEV)), b.to(DEV)
    for shape in ((4, 4, k), (16, 1, k), (1, 16, k), (5, 130, k)):
        x = features(shape, 2, 5).to(DEV)
        want = G.int8_linear(x.reshape(-1, k), wq.q, wq.scale, bd, leaky=True).reshape(shape[:2] + (33,))
        apart = torch.zeros(shape[0], shape[1] + 2, k, device=DEV)
        apart[:, :shape[1]] = x
        for y in (x, x.transpose(0, 1).contiguous().transpose(0, 1), apart[:, :shape[1]], apart[:, :shape[1]].contiguous()):
            assert torch.equal(G.int8_linear(y, wq.q, wq.scale, bd, leaky=True), want)

    def largest(x):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        G.int8_linear(x, wq.q, wq.scale, bd)
        return torch.cuda.max_memory_allocated() - before

    x = features((16, k), 1, 6).to(DEV)
    assert largest(x.reshape(4, 4, k)) == largest(x) < largest(torch.zeros(4, 5, k, device=DEV)[:, :4])


@gpu
def test_linear_special_values():
    """Zero rows give act(bias); a row with Inf / NaN gives NaN and leaves its neighbours alone; fp16 outputs overflow to Inf."""
    for n, k, o in ((4, 100, 40), (300, 100, 40)):
        x = torch.randn(n, k, generator=gen(1))
        x[0], x[1, 7], x[2, 99] = 0, math.nan, -math.inf
        w, b = weights(o, k, 3)
        wq = G.quantize_rows(w.to(DEV))
        y = G.int8_linear(x.to(DEV), wq.q, wq.scale, b.to(DEV), leaky=True)
        ref, bound = linear_ref_of(x, wq.q, wq.scale, b, True)
        assert bool(torch.isnan(ref[1:3]).all())
        assert_linear(y, ref, bound)
        assert torch.equal(y[0].cpu(), torch.where(b > 0, b, b * 0.2))
        h = G.int8_linear((x * 1e6).to(DEV), wq.q, wq.scale, out_dtype=torch.float16).cpu()
        ref, _ = linear_ref_of(x * 1e6, wq.q, wq.scale, None, False)
        over = ref.abs() > 65600
        assert bool(over.any()) and bool((h.double()[over] == ref[over].sign() * math.inf).all())


@gpu
@pytest.mark.parametrize("k", [100, 700])
def test_linear_scales_at_the_ends_of_the_range(k):
    """Results in range whose sum * x_scale is not: rows up to fp32's largest value times small weights, and 8-bit rows with scales of any
    size.  The epilogue moves a power of two between the scales; every kernel, both layouts."""
    tiny = torch.tensor([2.0 ** -149, 2.0 ** -127, 3.1e-39, 2.0 ** -107, 1.0, 2.0 ** 90, 2.0 ** 97, 1.7e38], dtype=torch.float32)
    for n, o in ((4, 24), (40, 150), (300, 40), (700, 260), (1100, 700)):
        x = torch.randn(n, k, generator=gen(n)).clamp(-3.3, 3.3)
        x = x * torch.tensor([1e38, 1e37, 1e30, 1.0])[torch.arange(n) % 4].unsqueeze(1)
        w, b = weights(o, k, 3)
        w = w * torch.tensor([2.0 ** -12, 2.0 ** -100, 2.0 ** -40])[torch.arange(o) % 3].unsqueeze(1)
        wq = G.quantize_rows(w.to(DEV))
        ref, bound = linear_ref_of(x, wq.q, wq.scale, b, True)
        assert bool((ref.abs() < 1e38).all()) and bool(((ref_rows(x)[0] @ wq.q.cpu().double().t()).abs() * ref_rows(x)[1].double()[:, None] > 1e39).any())
        y = G.int8_linear(x.to(DEV), wq.q, wq.scale, b.to(DEV), leaky=True)
        assert_linear(y, ref, bound)
        y = G.int8_linear(x.t().contiguous()[None].to(DEV), wq.q, wq.scale, b.to(DEV), leaky=True, channels_first=True)
        assert_linear(y[0].t(), ref, bound)

        q, s = ref_rows(torch.randn(n, k, generator=gen(n + 1)))
        s = tiny[torch.arange(n) % len(tiny)]
        ws = tiny.flip(0)[torch.arange(o) % len(tiny)]
        xq = q.to(torch.int8).to(DEV)
        for bias in (None, b):
            ref, bound = ref_linear(q, s, wq.q, ws, bias, False)
            y = G.int8_linear(xq, wq.q, ws.to(DEV), None if bias is None else bias.to(DEV), x_scale=s.to(DEV))
            assert_linear(y, ref, bound)
            y = G.int8_linear(xq[None], wq.q, ws.to(DEV), None if bias is None else bias.to(DEV), x_scale=s[None].to(DEV), channels_first=True)
            assert_linear(y[0].t(), ref, bound)


@gpu
def test_linear_output_beyond_32_bits():
    """More than 2^32 bytes of y: the rows at its end."""
    n, k, o = 1 << 20, 16, 2112
    x = features((n, k), 1, 4, torch.bfloat16).to(DEV)
    w, b = weights(o, k, 4)
    wq = G.quantize_rows(w.to(DEV))
    y = G.int8_linear(x, wq.q, wq.scale, b.to(DEV), out_dtype=torch.bfloat16)
    assert y.numel() * 2 > 2 ** 32
    for rows in (slice(0, 70), slice(n // 2 + 3, n // 2 + 70), slice(n - 70, n)):
        ref, bound = linear_ref_of(x[rows], wq.q, wq.scale, b, False)
        assert_linear(y[rows], ref, bound)


# ---- GPU: together, captured, on other streams, through both bindings ------------------------------------------------------------
def _together(q, scale, write, read, maps, layers):
    """Maps into the cache; the cached rows through the first layer; its output through the second; the maps read back."""
    (w1, s1, b1), (w2, s2, b2) = layers
    G.write_featmaps(q, scale, write, maps)
    h = G.int8_linear(q, w1, s1, b1, x_scale=scale, slots=read, leaky=True, out_dtype=torch.bfloat16)
    y = G.int8_linear(h, w2, s2, b2, leaky=True)
    return h, y, G.read_featmaps(q, scale, read)


def _layers(c):
    out = []
    for o, k, seed in ((2 * c, c, 1), (c + 3, 2 * c, 2)):
        w, b = weights(o, k, seed)
        r = G.quantize_rows(w.to(DEV))
        out.append((r.q, r.scale, b.to(DEV)))
    return out


@gpu
def test_operators_together():
    c, p = 66, 90
    store, q, scale = new_cache(6, p, c)
    maps = features((2, c, p), 1, 3).to(DEV)
    layers = _layers(c)
    read = torch.tensor([4, 2, 0], device=DEV)
    h, y, back = _together(q, scale, torch.tensor([2, 4], device=DEV), read, maps, layers)
    qc, sc = q[read].cpu(), scale[read].cpu()
    assert torch.equal(qc[1].double(), ref_rows(maps[0].t())[0])
    ref, bound = ref_linear(qc, sc, *layers[0], True)
    assert_linear(h, ref, bound)
    ref, bound = linear_ref_of(h, *layers[1], True)                           # from the operator's own bf16 rows: one answer
    assert_linear(y, ref, bound)
    assert torch.equal(back.cpu(), (qc.float() * sc.unsqueeze(-1)).transpose(1, 2))


@gpu
def test_captured_and_replayed():
    """The run above as two HIP graphs over the same cache, replayed in turn with eager calls between them: every replay equals the eager result
    on the inputs it saw (buffers are read and written in place, nothing is kept from the capture)."""
    c, p = 66, 90
    store, q, scale = new_cache(6, p, c)
    layers = _layers(c)
    inputs = [features((2, c, p), 1, 20 + i).to(DEV) for i in range(4)]
    static = [inputs[0].clone(), inputs[1].clone()]
    write = [torch.tensor([2, 4], device=DEV), torch.tensor([1, 4], device=DEV)]
    read = torch.tensor([4, 2, 1], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            _together(q, scale, write[i], read, static[i], layers)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_together(q, scale, write[i], read, static[i], layers))
        graphs.append(g)
    for turn in range(4):
        for i in range(2):
            x = inputs[(turn + 2 * i) % 4]
            static[i].copy_(x)
            graphs[i].replay()
            got = [t.clone() for t in outs[i]]
            torch.cuda.synchronize()
            q2, s2 = q.clone(), scale.clone()
            want = _together(int8._pitched(q2), s2, write[i], read, x, layers)
            for a, b in zip(got, want):
                assert torch.equal(a, b), (turn, i)


@gpu
def test_other_streams():
    """Two calls at once on two streams, with their own outputs and workspaces."""
    w, b = weights(300, 200, 7)
    wq = G.quantize_rows(w.to(DEV))
    xs = [features((3000 + i, 200), 1, 50 + i).to(DEV) for i in range(2)]
    want = [G.int8_linear(x, wq.q, wq.scale, b.to(DEV)) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(G.int8_linear(xs[i], wq.q, wq.scale, b.to(DEV)))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@gpu
def test_two_bindings_agree(monkeypatch):
    """The C++ extension and ctypes call the same C entries: equal bits, equal shapes, equal refusals."""
    assert _torch_ext.load(required=True) is not None
    c, p = 45, 70
    maps = features((2, c, p), 1, 3, torch.float16).to(DEV)
    w, b = weights(50, c, 2)
    slots = torch.tensor([2, 0], device=DEV)
    res = []
    for binding in ("torch_ext", "ctypes"):
        monkeypatch.setenv("GNR_BINDING", binding)
        store, q, scale = new_cache(3, p, c)
        wq = G.quantize_rows(w.to(DEV))
        G.write_featmaps(q, scale, slots, maps)
        m = G.quantize_rows(maps, channels_first=True)
        res.append([store, scale, wq.q, wq.scale, m.q, m.scale, G.read_featmaps(q, scale, slots, torch.bfloat16),
                    G.int8_linear(q, wq.q, wq.scale, b.to(DEV), x_scale=scale, slots=slots, channels_first=True),
                    G.int8_linear(maps, wq.q, wq.scale, b.to(DEV), leaky=True, channels_first=True, out_dtype=torch.float16),
                    G.int8_linear(w.to(DEV), wq.q, wq.scale), G.int8_linear(w.to(DEV)[0], wq.q, wq.scale),
                    G.int8_linear(wq.q, wq.q, wq.scale, x_scale=wq.scale), G.quantize_rows(maps.view(2, 5, 9, p)).q])
        with pytest.raises(ValueError):
            G.int8_linear(w.to(DEV)[:, 1:], wq.q, wq.scale)
        with pytest.raises(TypeError):
            G.write_featmaps(q, scale, slots.int(), maps)
    for i, (a, b) in enumerate(zip(*res)):
        assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b), i


@gpu
@pytest.mark.parametrize("binding, poison", [("ctypes", False), ("torch_ext", True)])
def test_under_guard_bands(binding, poison):
    """Random shapes with every device buffer fenced by 1 MiB of a known pattern (and, poisoned, full of 0xFF bytes: what lies between and
    behind rows must not count, and no workspace is read before it is written)."""
    from test_guard_bands import _guarded
    d = _guarded("int8", "--binding", binding, "--cases", "25", "--seed", "7" if poison else "8", *(["--poison"] if poison else []))
    assert d["ok"] and d["violations"] == 0, (d["report"], d["cases"])
    assert d["calls_checked"] >= 25 * 6


def test_m0_is_put_back():
    """Inline assembly that writes m0 (a reserved register: the compiler takes no clobber for it) saves it first and restores it last."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.abspath(G.__file__)), "csrc")
    found = 0
    for name in ("gnr_int8.hip", "gnr_int8.h", "gnr_quant.hip", "gnr_upsample8.hip"):
        text = open(os.path.join(csrc, name)).read()
        for block in re.findall(r'asm\s+volatile\s*\(\s*"([^"]*)"', text):
            steps = block.split("\\n\\t")
            if any(re.match(r"s_mov_b32 m0,", s) for s in steps):
                found += 1
                assert re.match(r"s_mov_b32 %0, m0$", steps[0]) and re.match(r"s_mov_b32 m0, %0$", steps[-1]), (name, block)
    assert found
