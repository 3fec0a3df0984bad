"""The upsampler in 8 bits (gazenerf_amd.upsample8) against a plain implementation that rounds where the definition says so.

Up to the last block's output every value has ONE answer and is computed here on the CPU exactly as defined: 8-bit rows (sums of whole
numbers, exact), an epilogue of named fp32 roundings, bf16 activations, a blur whose weights are powers of two in a fixed order.  What is
left for a tolerance is the RGB branch: fp32 sums of C products in an order of their own (u = 2^-24: at most (C + 3) u of the sum of
magnitudes), the upsampling of the running image (bilinear and blur: fewer than 16 roundings of a convex combination per level), and
the sigmoid (slope at most 1/4, expf and the quotient within 4 u of a value below 1)."""
import copy
import ctypes as C
import pickle
import sys
import threading

import pytest
import torch
import torch.nn.functional as F

import gazenerf_amd as G
from gazenerf_amd import _lib, upsample8
from gazenerf_amd.upsample import _channels, _expected_shapes, renderer_param_names
from test_int8 import DEV, features, gen, ref_rows

gpu = pytest.mark.gpu
U = 2.0 ** -24


def make_params(feat_nc, n_blocks, min_feat, seed, device=DEV):
    g = gen(seed)
    out = {}
    for base, (o, k) in _expected_shapes(feat_nc, n_blocks, min_feat).items():
        out[base + ".weight"] = (torch.randn(o, k, 1, 1, generator=g) * (2.0 / (o + k)) ** 0.5 * 1.5).to(device)
        out[base + ".bias"] = (torch.randn(o, generator=g) * 0.1).to(device)
    return {n: out[n] for n in renderer_param_names(n_blocks)}


def product(q, s, w, b):
    """fp32 roundings of the epilogue: fl(fl(sum) * s), one fused multiply-add, the leaky product; then bf16.  q, w whole numbers in float64."""
    wq, ws = ref_rows(w.reshape(w.shape[0], -1))
    t = (q @ wq.t()).float() * s.unsqueeze(-1)
    v = (t.double() * ws.double() + b.cpu().double()).float()
    return torch.maximum(v, v * torch.tensor(0.2)).bfloat16()


def up_image(rgb):
    """blur(bilinear x2) of [B, 3, S, S] in 64 bits."""
    x = F.interpolate(rgb, scale_factor=2, mode="bilinear", align_corners=False)
    x = F.pad(x, (1, 1, 1, 1), mode="reflect")
    k = torch.tensor([1.0, 2.0, 1.0], dtype=x.dtype)
    k = (k[:, None] * k[None, :] / 16).view(1, 1, 3, 3).expand(3, 1, 3, 3)
    return F.conv2d(x, k, groups=3)


def reference(rows, scale, params, S, n_blocks, min_feat, final):
    """rows float64 [B, P, C], scale float32 [B, P] -> (image float64, bound)."""
    B, P, Cn = rows.shape
    ch = _channels(Cn, n_blocks, min_feat)
    get = lambda n: params[n].detach().cpu()

    def rgb_conv(v, level):
        w, b = get("feat_2_rgb_list.%d.weight" % level).reshape(3, -1).double(), get("feat_2_rgb_list.%d.bias" % level).double()
        y = v.double() @ w.t() + b
        mag = v.double().abs() @ w.abs().t() + b.abs()
        s = int(round(v.shape[1] ** 0.5))
        shape = lambda t: t.transpose(1, 2).reshape(B, 3, s, s)
        return shape(y), shape((v.shape[2] + 3) * U * mag)

    q, s = rows, scale
    res = None                                                              # None: the 8-bit rows are the residual
    rgb, err = rgb_conv((rows.float() * scale.unsqueeze(-1)), 0)
    rgb, err = up_image(rgb), up_image(err) + 16 * U * up_image(rgb.abs())
    for i in range(n_blocks):
        c = ch[i]
        a1 = product(q, s, get("feat_upsample_list.%d.layer_1.weight" % i), get("feat_upsample_list.%d.layer_1.bias" % i))
        a2 = product(*ref_rows(a1.float()), get("feat_upsample_list.%d.layer_2.weight" % i), get("feat_upsample_list.%d.layer_2.bias" % i))
        idx = torch.arange(4 * c) % c
        if res is None:
            u = (q[..., idx] * s.double().unsqueeze(-1) + a2.double()).float()    # one fused multiply-add
        else:
            u = a2.float() + res.float()[..., idx]
        u = u.reshape(B, S, S, c, 2, 2).permute(0, 3, 1, 4, 2, 5).reshape(B, c, 2 * S, 2 * S)
        pad = F.pad(u, (1, 1, 1, 1), mode="reflect")
        rowsum = (0.25 * pad[:, :, :-2] + 0.5 * pad[:, :, 1:-1]) + 0.25 * pad[:, :, 2:]
        v = (0.25 * rowsum[..., :-2] + 0.5 * rowsum[..., 1:-1]) + 0.25 * rowsum[..., 2:]
        S *= 2
        v = v.permute(0, 2, 3, 1).reshape(B, S * S, c)
        net = product(*ref_rows(v), get("feat_layers.%d.weight" % i), get("feat_layers.%d.bias" % i))
        y, e = rgb_conv(net, i + 1)
        rgb, err = rgb + y, err + e + U * (rgb.abs() + y.abs())
        if i < n_blocks - 1:
            rgb, err = up_image(rgb), up_image(err) + 16 * U * up_image(rgb.abs())
            q, s = ref_rows(net.float())
            res = net
    if final:
        rgb, err = torch.sigmoid(rgb), err / 4 + 4 * U
    return rgb, err


def check(img, rows, scale, params, S, n_blocks, min_feat, final):
    ref, err = reference(rows, scale, params, S, n_blocks, min_feat, final)
    assert img.shape == ref.shape
    d = (img.cpu().double() - ref).abs()
    bad = d > err
    assert not bool(bad.any()), (int(bad.sum()), float((d / err).max()))


# channels that a residual's four values wrap around in, one and several groups of threads a workgroup, rows of more channels than threads
CASES = [(6, 2, 4, 16, 2, True), (33, 1, 8, 16, 1, False), (64, 2, 32, 16, 1, True), (129, 1, 32, 32, 2, True), (258, 2, 32, 16, 1, False),
         (330, 1, 32, 16, 1, True), (1024, 1, 32, 16, 1, True), (48, 4, 8, 16, 1, True), (258, 3, 32, 64, 1, True)]


@gpu
@pytest.mark.parametrize("feat_nc, n_blocks, min_feat, S, B, final", CASES)
def test_image_from_a_map(feat_nc, n_blocks, min_feat, S, B, final):
    params = make_params(feat_nc, n_blocks, min_feat, feat_nc)
    x = features((B, feat_nc, S, S), 1, feat_nc + S).to(DEV)
    with torch.no_grad():
        img = G.neural_render_int8(x, params, n_blocks, min_feat, final)
    q, s = ref_rows(x.flatten(2).transpose(1, 2))
    check(img, q, s, params, S, n_blocks, min_feat, final)


def plain_network(x, params, n_blocks, min_feat, half):
    """The network on x [B, C, S, S] in 64 bits -> the image before the sigmoid.  ``half`` > 0: where the definition rounds rows or weights to 8
    bits, an error of its own, uniform in +- half a step, for every value."""
    B, Cn, S, _ = x.shape
    g = gen(17)

    def row(t):
        return t + (torch.rand(t.shape, generator=g, dtype=torch.float64) * 2 - 1) * half * (t.abs().amax(-1, keepdim=True) / 127) if half else t

    def conv(t, name):
        w = params[name + ".weight"].detach().cpu().double().reshape(-1, t.shape[-1])
        y = t @ row(w).t() + params[name + ".bias"].detach().cpu().double()
        return torch.maximum(y, 0.2 * y)

    def rgb_conv(t, level):
        w = params["feat_2_rgb_list.%d.weight" % level].detach().cpu().double().reshape(3, -1)
        y = t @ w.t() + params["feat_2_rgb_list.%d.bias" % level].detach().cpu().double()
        return y.transpose(1, 2).reshape(B, 3, S, S)

    net = row(x.cpu().double().flatten(2).transpose(1, 2))
    res, rgb = net, up_image(rgb_conv(net, 0))
    for i in range(n_blocks):
        c = net.shape[-1]
        a2 = conv(row(conv(net, "feat_upsample_list.%d.layer_1" % i)), "feat_upsample_list.%d.layer_2" % i)
        u = a2 + res[..., torch.arange(4 * c) % c]
        u = u.reshape(B, S, S, c, 2, 2).permute(0, 3, 1, 4, 2, 5).reshape(B * c, 1, 2 * S, 2 * S)
        k = torch.tensor([0.25, 0.5, 0.25], dtype=torch.float64)
        v = F.conv2d(F.pad(u, (1, 1, 1, 1), mode="reflect"), (k[:, None] * k[None, :])[None, None])
        S *= 2
        net = conv(row(v.reshape(B, c, S * S).transpose(1, 2)), "feat_layers.%d" % i)
        rgb, res = rgb + rgb_conv(net, i + 1), net
        if i < n_blocks - 1:
            rgb, net = up_image(rgb), row(net)
    return rgb


@gpu
@pytest.mark.parametrize("feat_nc, n_blocks, min_feat, B", [(36, 2, 8, 2), (258, 3, 32, 1)])
def test_the_8_bit_image_is_as_near_to_the_fp32_one_as_rounding_says(feat_nc, n_blocks, min_feat, B):
    """What 8 bits cost: the rms difference to the fp32 renderer's image against that of the network in 64 bits with an independent error, uniform
    in +- half a step, at every 8-bit rounding.  Rounding errors are as large as that and nearly independent; two of them that were not would
    add up to at most twice the rms.  (bf16 between the products adds 2^-9 of a value where 8 bits add 2^-8 of the row's largest: inside.)"""
    params = make_params(feat_nc, n_blocks, min_feat, feat_nc + 1)
    x = features((B, feat_nc, 16, 16), 1, feat_nc).to(DEV)
    rms = lambda t: float(t.double().pow(2).mean().sqrt())
    with torch.no_grad():
        exact = G.neural_render(x, params, n_blocks, min_feat, False).cpu().double()
        d = rms(G.neural_render_int8(x, params, n_blocks, min_feat, False).cpu().double() - exact)
    plain = plain_network(x, params, n_blocks, min_feat, 0.0)
    model = rms(plain_network(x, params, n_blocks, min_feat, 1.0 / 2) - plain)
    print("8-bit rms error %.3e, of independent roundings %.3e, image rms %.3e" % (d, model, rms(exact)))
    assert rms(exact - plain) < 1e-4 * rms(plain)                    # the same network
    assert d <= 2 * model and model < 0.1 * rms(plain)


@gpu
def test_image_from_cached_rows():
    """The same bits from the slots of a cache; padding slots are zero maps, slots outside the cache NaN images."""
    params = make_params(33, 2, 8, 3)
    x = features((3, 33, 16, 16), 1, 5).to(DEV)
    cache = G.FeatureMapCache(5, 33, 256, device=DEV)
    cache.write([4, 0, 2], x)
    with torch.no_grad():
        direct = G.neural_render_int8(x, params, 2, 8)
        slots = torch.tensor([2, -1, 4, 5, 0, 2], device=DEV)
        img = G.neural_render_int8(None, params, 2, 8, cache=cache, slots=slots)
        zero = G.neural_render_int8(torch.zeros_like(x[:1]), params, 2, 8)
        never = G.neural_render_int8(None, params, 2, 8, cache=cache, slots=torch.tensor([1], device=DEV))
        view = G.FeatureMapCache(5, 33, 256, device=DEV)                         # rows the product cannot read in place
        view.q, view.scale = cache.q.clone()[..., :33].contiguous(), cache.scale
        odd = G.neural_render_int8(None, params, 2, 8, cache=view, slots=slots)
    assert torch.equal(img[[0, 2, 4, 5]], direct[[2, 0, 1, 2]]) and torch.equal(img[1], zero[0])
    assert bool(torch.isnan(img[3]).all()) and bool(torch.isnan(never).all())
    assert torch.equal(odd.nan_to_num(), img.nan_to_num())


def small_renderer(device=DEV, **kw):
    torch.manual_seed(0)
    return G.NeuralRendererAMD(feat_nc=36, featmap_size=16, img_size=64, min_feat=8, **kw).to(device)


@gpu
def test_module_replays_and_follows_its_parameters():
    """graph_inference: every replay equals the eager call on the inputs and parameters it saw -- after an in-place update (an optimizer's), a
    new storage, a load_state_dict -- with eager calls in between and two input shapes alive."""
    net = small_renderer(precision="int8")
    eager = lambda x: G.neural_render_int8(x, {k: v for k, v in net.named_parameters() if k != "bg_featmap"}, 2, 8)
    xs = [features((b, 36, 16, 16), 1, b).to(DEV) for b in (1, 2, 1, 2, 1)]
    with torch.no_grad():
        for x in xs:
            assert torch.equal(net(x), eager(x))
        graphed = net._int8(torch.device(DEV, torch.cuda.current_device()))
        assert graphed.captures == 2 and graphed.replays == 5 and graphed.weights.quantised == 1
        before = net(xs[0])
        net.feat_layers[0].weight.mul_(1.5)                                     # counted by torch
        net.feat_2_rgb_list[1].bias.add_(0.25)                                  # read in place by the graph
        for x in xs[:3]:
            assert torch.equal(net(x), eager(x))
        assert not torch.equal(net(xs[0]), before) and graphed.weights.quantised == 2 and graphed.captures == 2
        state = {k: v * 0.5 for k, v in net.state_dict().items()}
        net.load_state_dict(state)
        assert torch.equal(net(xs[0]), eager(xs[0]))
        net.feat_layers[1].weight.data.copy_(net.feat_layers[1].weight.data * 2)   # not counted: train() / eval() looks again
        net.eval()
        assert torch.equal(net(xs[1]), eager(xs[1]))
        twin = copy.deepcopy(net)
        assert torch.equal(twin(xs[0]), net(xs[0])) and twin._int8 is not net._int8
    with torch.inference_mode():
        assert torch.equal(net(xs[3]), eager(xs[3]))


@gpu
def test_module_on_two_streams_at_once():
    net = small_renderer(precision="int8")
    xs = [features((2, 36, 16, 16), 1, 40 + i).to(DEV) for i in range(2)]
    with torch.no_grad():
        want = [net(x) for x in xs]
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in xs], [[], []]
        for turn in range(6):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(net(xs[(i + turn) % 2]))
        torch.cuda.synchronize()
    assert all(torch.equal(got[i][turn], want[(i + turn) % 2]) for i in range(2) for turn in range(6))
    assert len(net._int8.streams) == 3


def in_threads(n, work):
    """work(i) in n threads at once, with the interpreter switching between them as often as it can; their results in order."""
    out, errors, start = [None] * n, [], threading.Barrier(n)

    def body(i):
        try:
            start.wait()
            out[i] = work(i)
        except BaseException as e:
            errors.append(e)
    every = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=body, args=(i,)) for i in range(n)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(every)
    if errors:
        raise errors[0]
    return out


def test_replays_of_two_threads_stay_apart():
    """The replay's own steps -- copy in, replay, copy out -- with a stand-in for the graph and its tensors on the CPU: each thread gets what
    belongs to its input."""
    class Replay:
        def __init__(self, static, img):
            self.static, self.img = static, img

        def replay(self):
            self.img.copy_(self.static * 2)

    class OnCpu(upsample8.GraphedUpsample8):
        def _capture(self, params, n_blocks, min_feat, final_actvn, x, cache, slots):
            static, call = torch.empty_like(x), type("Call", (), {"img": torch.empty_like(x)})()
            self.captures += 1
            return Replay(static, call.img), static, call

    class NoWeights(upsample8.Int8Weights):
        def refresh(self, params, n_blocks):
            pass

    graphed = OnCpu(NoWeights())
    params = {n: torch.zeros(1) for n in renderer_param_names(1)}

    def work(i):
        x = torch.full((4,), float(i + 1))
        return sum(not torch.equal(graphed(params, 1, 8, True, x=x), 2 * x) for _ in range(3000))
    assert in_threads(2, work) == [0, 0] and graphed.captures == 1


def test_weights_copy_empty():
    """Int8Weights and its lock: copies and pickles start empty."""
    w = upsample8.Int8Weights()
    w.quantised, w.rows["x"] = 3, None
    for twin in (copy.deepcopy(w), pickle.loads(pickle.dumps(w))):
        assert not twin.rows and twin.seen is None and twin.quantised == 0 and twin.lock is not w.lock


def test_more_streams_than_renderers(monkeypatch):
    """Streams used in turn keep what they have: the fifth of five gets none, instead of taking the place of one that is about to come back.
    A stream that is not used any more makes room in the end."""
    now = type("Stream", (), {})()
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: now)
    renderers, dev = upsample8.Int8Renderers(), torch.device("cuda", 0)

    def on(handle):
        now.cuda_stream = handle
        return renderers(dev)
    first = [on(h) for h in range(5)]
    assert all(r is not None for r in first[:4]) and len(set(map(id, first))) == 5 and first[4] is None
    for _ in range(20):
        assert [on(h) for h in range(5)] == first
    assert [on(4) for _ in range(40)][-1] is not None and len(renderers.streams) == 4     # the other four fell silent
    assert sum(on(h) is None for h in range(5)) == 1
    assert upsample8.Int8Renderers(0)(dev) is None                                        # none kept: every call without a graph


@gpu
def test_module_on_more_streams_than_it_keeps_graphs_for():
    """Six streams in turn: four graphs, captured once; the images are right on all of them, after a change of the weights too."""
    net = small_renderer(precision="int8")
    x = features((1, 36, 16, 16), 1, 90).to(DEV)
    params = {k: v for k, v in net.named_parameters() if k != "bg_featmap"}
    streams = [torch.cuda.Stream() for _ in range(6)]
    with torch.no_grad():
        for turn in range(4):
            want = G.neural_render_int8(x, params, 2, 8)
            torch.cuda.synchronize()
            got = []
            for s in streams:
                with torch.cuda.stream(s):
                    got.append(net(x))
            torch.cuda.synchronize()
            assert all(torch.equal(g, want) for g in got)
            net.feat_layers[0].weight.mul_(1.25)
            torch.cuda.synchronize()
    kept = list(net._int8.streams.values.values())
    assert len(kept) == 4 and all(r.captures == 1 and r.replays == 4 and r.weights.quantised == 4 for r in kept)


@gpu
def test_more_batch_sizes_than_graphs():
    net = small_renderer(precision="int8")
    xs = [features((b, 36, 16, 16), 1, b).to(DEV) for b in range(1, 7)]
    params = {k: v for k, v in net.named_parameters() if k != "bg_featmap"}
    with torch.no_grad():
        want = [G.neural_render_int8(x, params, 2, 8) for x in xs]
        for _ in range(3):
            assert all(torch.equal(net(x), w) for x, w in zip(xs, want))
    graphed = net._int8(torch.device(DEV, torch.cuda.current_device()))
    assert graphed.captures == 4 and graphed.replays == 12 and graphed.weights.quantised == 1


@gpu
def test_a_graph_does_not_keep_a_cache():
    """A deleted FeatureMapCache gives its memory back, although a graph that read it is still there."""
    net = small_renderer()
    x = features((2, 36, 16, 16), 1, 91).to(DEV)
    cache = G.FeatureMapCache(2000, 36, 256, device=DEV)
    cache.write([0, 1], x)
    with torch.no_grad():
        want = net.render_cached(cache, [1, 0])
    torch.cuda.synchronize()
    held, size = torch.cuda.memory_allocated(), cache.q.untyped_storage().nbytes() + cache.scale.untyped_storage().nbytes()
    del cache
    assert held - torch.cuda.memory_allocated() >= size
    again = G.FeatureMapCache(2000, 36, 256, device=DEV)                          # likely where the first one stood: the graph reads it in place
    again.write([0, 1], x.flip(0))
    with torch.no_grad():
        assert torch.equal(net.render_cached(again, [0, 1]), want)


@gpu
@pytest.mark.parametrize("own_streams", [False, True])
def test_module_in_threads(own_streams):
    """Three threads, each with its own map, on the default stream and on streams of their own; the graphs are captured while the others run."""
    net = small_renderer(precision="int8")
    xs = [features((1 + (i == 2), 36, 16, 16), 1, 70 + i).to(DEV) for i in range(3)]
    params = {k: v for k, v in net.named_parameters() if k != "bg_featmap"}
    with torch.no_grad():
        want = [G.neural_render_int8(x, params, 2, 8) for x in xs]
    torch.cuda.synchronize()

    def work(i):
        with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream() if own_streams else torch.cuda.current_stream()):
            got = [net(xs[i]) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
        return all(torch.equal(g, want[i]) for g in got)
    assert in_threads(3, work) == [True] * 3


@gpu
@pytest.mark.parametrize("warm", [False, True])
def test_module_captured_by_a_caller(warm):
    """The caller's own graph quantises the weights: replays follow an in-place update, and an eager call before the first replay does not
    take weights that were only recorded."""
    net = small_renderer(precision="int8")
    static, xs = features((1, 36, 16, 16), 1, 50).to(DEV), [features((1, 36, 16, 16), 1, 51 + i).to(DEV) for i in range(3)]
    eager = lambda x: G.neural_render_int8(x, {k: v for k, v in net.named_parameters() if k != "bg_featmap"}, 2, 8)
    with torch.no_grad():
        want = eager(xs[0])                                                     # the library is loaded
        if warm:
            net(static)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = net(static)
        assert torch.equal(net(xs[0]), want)
        for turn in range(3):
            for x in xs:
                static.copy_(x)
                graph.replay()
                got = out.clone()
                torch.cuda.synchronize()
                assert torch.equal(got, eager(x)) and torch.equal(net(x), got)
            net.feat_upsample_list[0].layer_1.weight.mul_(1.25)


@gpu
def test_module_made_in_inference_mode():
    """Writes to tensors made in inference mode are not counted: the weights are quantised in every call."""
    with torch.inference_mode():
        net = small_renderer(precision="int8")
        x = features((1, 36, 16, 16), 1, 60).to(DEV)
        for _ in range(2):
            assert torch.equal(net(x), G.neural_render_int8(x, {k: v for k, v in net.named_parameters() if k != "bg_featmap"}, 2, 8))
            net.feat_layers[0].weight.mul_(1.5)


def test_module_copies():
    """Copies and pickles start without captured graphs; a module pickled before there was a precision is an fp32 one."""
    net = small_renderer("cpu", precision="int8")
    for twin in (copy.deepcopy(net), pickle.loads(pickle.dumps(net))):
        assert twin.precision == "int8" and not twin._int8.streams and twin._int8 is not net._int8
    state = dict(net.__dict__)
    del state["precision"], state["_int8"]
    old = G.NeuralRendererAMD.__new__(G.NeuralRendererAMD)
    old.__setstate__(state)
    assert old.precision == "fp32" and not old._int8.streams and old.eval() is old


@gpu
@pytest.mark.parametrize("precision", ["fp32", "int8"])
def test_module_refuses_a_tangent(precision):
    """A dual input or weight under no_grad, where a graph would be replayed: refused, not returned without its tangent."""
    from torch.autograd import forward_ad
    net = small_renderer(precision=precision)
    x = features((1, 36, 16, 16), 1, 80).to(DEV)
    with torch.no_grad():
        want = net(x)
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode gradient|forward mode AD"):
                net(forward_ad.make_dual(x, torch.ones_like(x)))
            assert torch.equal(net(x), want)
            name, p = "feat_layers.0.weight", net.feat_layers[0].weight.detach()
            with pytest.raises(RuntimeError, match="forward-mode gradient|forward mode AD"):
                torch.func.functional_call(net, {name: forward_ad.make_dual(p, torch.ones_like(p))}, (x,))
        assert torch.equal(net(x), want)


@gpu
def test_module_renders_cached_views():
    net = small_renderer()                                                       # fp32 by itself; cached views are 8-bit
    x = features((3, 36, 16, 16), 1, 9).to(DEV)
    cache = G.FeatureMapCache(4, 36, 256, device=DEV)
    cache.write([0, 1, 3], x)
    params = {k: v for k, v in net.named_parameters() if k != "bg_featmap"}
    with torch.no_grad():
        want = G.neural_render_int8(x, params, 2, 8)
        for slots in ([3, 0], 1, torch.tensor([0, 3], device=DEV), [0, 1]):
            img = net.render_cached(cache, slots)
            idx = {0: 0, 1: 1, 3: 2}
            assert torch.equal(img, want[[idx[int(s)] for s in cache.slots(slots)]])
        cache.write(1, x[:1])                                                    # the graph reads the cache in place
        assert torch.equal(net.render_cached(cache, [0, 1]), want[[0, 0]])
        with pytest.raises(IndexError):
            net.render_cached(cache, [4])
        with pytest.raises(ValueError, match="cache holds"):
            net.render_cached(G.FeatureMapCache(4, 35, 256, device=DEV), [0])
    with pytest.raises(RuntimeError, match="no backward"):
        net.render_cached(cache, [0])
    with pytest.raises(RuntimeError, match="no backward"):
        small_renderer(precision="int8")(x)


@gpu
def test_network_caches_and_renders_views():
    """GazeNeRFNetAMD: cache_views renders and keeps the merged maps, render_views turns them into the images of its own forward in 8 bits."""
    from gazenerf_amd import synth
    torch.manual_seed(1)
    net = G.GazeNeRFNetAMD(featmap_size=16, pred_img_size=32, num_sample_coarse=32, renderer_precision="int8").to(DEV)
    p = {k: v.to(DEV) for k, v in synth.synth_problem(16, batch=2, camera="3", seed=2).items()}
    args = dict(batch_xy=p["xy"], shape_code=p["shape_code"], appea_code=p["appea_code"], gaze_code=p["gaze"], batch_Rmats=p["R"], batch_Tvecs=p["T"],
                batch_inv_inmats=p["Kinv"])
    cache = G.FeatureMapCache(3, net.featmap_nc, 256, device=DEV)
    net.cache_views(cache, [2, 0], **args)
    img = net.render_views(cache, [0, 2, 0])
    with torch.no_grad():
        full = net("test", batch_uv=None, bg_code=None, **args)["coarse_dict"]
    assert torch.equal(img, full["merge_img"][[1, 0, 1]])
    assert bool(torch.isfinite(img).all())


# ---- CPU: refusals ---------------------------------------------------------------------------------------------------------------
def test_refusals(lib_built):
    with pytest.raises(ValueError, match="precision"):
        G.NeuralRendererAMD(precision="int4")
    net = G.NeuralRendererAMD(feat_nc=24, featmap_size=16, img_size=32, min_feat=8, precision="int8")
    with pytest.raises(RuntimeError, match="no backward"):
        net(torch.zeros(1, 24, 16, 16))
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA/ROCm"):
        net(torch.zeros(1, 24, 16, 16))
    params = {k: v for k, v in net.named_parameters() if k != "bg_featmap"}
    with torch.no_grad(), pytest.raises(ValueError, match="either a feature map or a cache"):
        G.neural_render_int8(None, params, 1, 8)
    cache = G.FeatureMapCache(2, 24, 256, device="cpu")
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA/ROCm"):
        G.neural_render_int8(None, params, 1, 8, cache=cache, slots=torch.zeros(1, dtype=torch.int64))


def test_c_entry_refuses(lib_built):
    lib = _lib.load()

    def args(prob={}, rows={}):
        p, q, w = _lib.GnrUpsampleProblem(), _lib.GnrUpsampleInt8(), _lib.GnrUpsampleWeights()
        p.batch, p.feat_nc, p.featmap_size, p.n_blocks, p.min_feat, p.final_sigmoid, p.x = 1, 24, 16, 1, 8, 1, 4096
        for s in ("up1", "up2", "feat"):
            getattr(q, s + "_w")[0], getattr(q, s + "_pitch")[0], getattr(q, s + "_s")[0] = 4096, 128, 4096
            getattr(w, s + "_b")[0] = 4096
        for i in range(2):
            w.rgb_w[i], w.rgb_b[i] = 4096, 4096
        for k, v in prob.items():
            setattr(p, k, v)
        for k, v in rows.items():
            setattr(q, k, v)
        return p, q, w

    cached = dict(x_q=4096, x_batch=8192, x_pitch=32, x_scale=4096, x_scale_batch=256)
    bad = [(dict(struct_size=3), {}, "struct_size"), ({}, dict(struct_size=3), "struct_size"), (dict(batch=0), {}, "batch"), (dict(featmap_size=24), {}, "power of two"),
           (dict(feat_nc=1025), {}, "1024"), (dict(x=None), {}, "x is NULL"), (dict(feat_nc=3, min_feat=1), {}, "at least 4"), ({}, cached, "both x and x_q"), (dict(batch=65536), {}, "65536"),
           (dict(x=None), dict(cached, x_scale=None), "x_scale"), (dict(x=None), dict(cached, x_pitch=24), "16-byte"), (dict(x=None), dict(cached, x_pitch=16), "16-byte"),
           (dict(x=None), dict(cached, x_q=4104), "16-byte"), (dict(x=None), dict(cached, slots=4096), "n_slots")]
    for prob, rows, word in bad:
        p, q, w = args(prob, rows)
        assert lib.gnr_upsample_int8_workspace_bytes(C.byref(p), C.byref(q)) == 0 and word in lib.gnr_last_error().decode(), (prob, rows, lib.gnr_last_error())
        assert lib.gnr_upsample_int8_fwd(C.byref(p), C.byref(w), C.byref(q), 4096, 4096, 1 << 30, None) != 0
    p, q, w = args()
    need = lib.gnr_upsample_int8_workspace_bytes(C.byref(p), C.byref(q))
    assert need > 0
    for a, word in (((C.byref(w), C.byref(q), None, 4096, need), "image"), ((None, C.byref(q), 4096, 4096, need), "weights"),
                    ((C.byref(w), C.byref(q), 4096, 4096, need - 1), "workspace"), ((C.byref(w), C.byref(q), 4096, 4104, need), "256-byte")):
        assert lib.gnr_upsample_int8_fwd(C.byref(p), *a, None) != 0 and word in lib.gnr_last_error().decode()
    for field in ("up1_w", "up2_s", "feat_w"):
        p, q, w = args()
        getattr(q, field)[0] = None
        assert lib.gnr_upsample_int8_fwd(C.byref(p), C.byref(w), C.byref(q), 4096, 4096, need, None) != 0
    p, q, w = args()
    w.rgb_b[1] = None
    assert lib.gnr_upsample_int8_fwd(C.byref(p), C.byref(w), C.byref(q), 4096, 4096, need, None) != 0
