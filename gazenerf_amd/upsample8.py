"""The upsampler in 8 bits, for inference: ``neural_render_int8`` and what ``NeuralRendererAMD(precision="int8")`` runs.

The network of ``gazenerf_amd.upsample`` (models/neural_renderer.py:100-113) with its 1x1 convolutions as 8-bit products
(``gazenerf_amd.int8``, one scale a pixel and one a channel), activations between them in bf16, the blur, the RGB branch and every
epilogue in fp32.  The feature map comes as a tensor [B, C, S, S] or as slots of a ``FeatureMapCache``, whose rows the first product
reads as they are; both give the same image bit for bit.  There is no backward.
"""
from __future__ import annotations

import ctypes as C
import threading
from typing import Dict, Optional

import torch

from . import _lib, int8
from .render import _check_tensor, _stream_ptr
from .upsample import RecentlyUsed, _expected_shapes, _weights_struct, capture_graph, renderer_param_names

_CONVS = (("up1", "feat_upsample_list.%d.layer_1"), ("up2", "feat_upsample_list.%d.layer_2"), ("feat", "feat_layers.%d"))


class Int8Weights:
    """The renderer's convolution weights as 8-bit rows, quantised once and again when a parameter changed: another tensor, a
    higher ``_version`` (torch counts every in-place write) or another ``data_ptr()``.  An in-place write through ``.data`` is invisible to
    all three, and so is one by a replayed graph: call ``clear()`` after one.  The buffers stay where they are while shapes and device do,
    so captured graphs that read them see the new values.  One per module and HIP stream (``Int8Renderers``); threads that share it
    hold ``lock`` from ``refresh`` until they have what they took from it."""

    def __init__(self):
        self.lock = threading.RLock()
        self.clear()

    def clear(self):
        self.rows: Dict[str, int8.QuantizedRows] = {}
        self.seen = None
        self.quantised = 0

    def __reduce__(self):                          # a copy or a pickle starts empty, with a lock of its own
        return Int8Weights, ()

    def refresh(self, params: Dict[str, torch.Tensor], n_blocks: int) -> None:
        names = [name % i for i in range(n_blocks) for _, name in _CONVS]
        flat = [params[n + ".weight"] for n in names]
        counted = not any(t.is_inference() for t in flat)       # torch counts no writes to tensors made in inference mode
        if counted and self.seen is not None and len(self.seen) == len(flat) and all(
                a is t and v == t._version and d == t.data_ptr() for (a, v, d), t in zip(self.seen, flat)):
            return
        self.seen = None                                        # a call that raises half-way leaves nothing that looks current
        for n, t in zip(names, flat):
            t2 = t.detach().reshape(t.shape[0], -1)
            old = self.rows.get(n)
            if old is None or old.q.shape != t2.shape or old.q.device != t2.device:
                q = int8.empty_rows(*t2.shape, device=t2.device)
                old = self.rows[n] = int8.QuantizedRows(q, torch.empty(t2.shape[0], dtype=torch.float32, device=t2.device))
            int8.quantize_rows_into(t2, old.q, old.scale)
        if counted:
            self.seen = [(t, t._version, t.data_ptr()) for t in flat]
        self.quantised += 1

    def fill(self, s: "_lib.GnrUpsampleInt8", n_blocks: int):
        for i in range(n_blocks):
            for short, name in _CONVS:
                r = self.rows[name % i]
                getattr(s, short + "_w")[i] = r.q.data_ptr()
                getattr(s, short + "_pitch")[i] = int8.row_pitch(r.q.shape[1])
                getattr(s, short + "_s")[i] = r.scale.data_ptr()


def _checked_params(params, C_in, n_blocks, min_feat, dev):
    out = {}
    shapes = _expected_shapes(C_in, n_blocks, min_feat)
    for name in renderer_param_names(n_blocks):
        t = params[name]
        _check_tensor(name, t)
        base = name.rsplit(".", 1)[0]
        want = shapes[base] if name.endswith(".weight") else (shapes[base][0],)
        t2 = t.detach().reshape(t.shape[0], -1) if name.endswith(".weight") else t.detach()
        if tuple(t2.shape) != want:
            raise ValueError("%s must have shape %s (+[1,1]), got %s" % (name, want, tuple(t.shape)))
        if t.device != dev:
            raise RuntimeError("%s lives on %s, the feature map on %s" % (name, t.device, dev))
        out[name] = t2.contiguous()
    return out


class _Call:
    """One ``gnr_upsample_int8_fwd``: the structs and every tensor they point into."""

    def __init__(self, params, weights: Int8Weights, n_blocks, min_feat, final_actvn, x=None, cache=None, slots=None):
        if (x is None) == (cache is None):
            raise ValueError("either a feature map or a cache with slots")
        if x is not None:
            _check_tensor("x", x)
            if x.dim() != 4 or x.shape[2] != x.shape[3]:
                raise ValueError("x must be [B, C, S, S], got %s" % (tuple(x.shape),))
            B, Cn, S, _ = x.shape
            dev = x.device
        else:
            int8._check_cache(cache.q, cache.scale, slots, None)
            int8._one_device(q=cache.q, scale=cache.scale, slots=slots)
            B, Cn, dev = slots.shape[0], cache.q.shape[2], cache.q.device
            S = int(round(cache.q.shape[1] ** 0.5))
            if S * S != cache.q.shape[1]:
                raise ValueError("the cache holds %d pixels a map: not a square" % cache.q.shape[1])
        if B < 1:
            raise ValueError("empty batch")
        self.params = _checked_params(params, Cn, n_blocks, min_feat, dev)
        self.p, self.s = _lib.GnrUpsampleProblem(), _lib.GnrUpsampleInt8()
        p, s = self.p, self.s
        with weights.lock:
            weights.refresh(params, n_blocks)
            weights.fill(s, n_blocks)
            self.rows = dict(weights.rows)
        p.batch, p.feat_nc, p.featmap_size, p.n_blocks, p.min_feat, p.final_sigmoid = B, Cn, S, n_blocks, min_feat, int(final_actvn)
        if x is not None:
            self.x = x.detach().contiguous()
            p.x = self.x.data_ptr()
        else:
            q = int8._pitched(cache.q)
            scale = cache.scale if cache.scale.stride(1) == 1 or cache.scale.shape[1] == 1 else cache.scale.contiguous()
            self.x, self.q, self.scale = slots.contiguous(), q, scale
            s.x_q, s.x_batch, s.x_pitch = q.data_ptr(), int8._stride(q, 0, 0), int8._stride(q, 1, int8.row_pitch(Cn))
            s.x_scale, s.x_scale_batch, s.slots, s.n_slots = scale.data_ptr(), int(scale.stride(0)), self.x.data_ptr(), q.shape[0]
        self.w = _weights_struct(self.params, n_blocks)
        self.dev = dev
        lib = _lib.load()
        need = lib.gnr_upsample_int8_workspace_bytes(C.byref(p), C.byref(s))
        if need == 0:
            _lib.check(1, lib)
        self.ws = torch.empty(int(need), dtype=torch.uint8, device=dev)
        self.img = torch.empty(B, 3, S << n_blocks, S << n_blocks, device=dev, dtype=torch.float32)

    def __call__(self):
        lib = _lib.load()
        with torch.cuda.device(self.dev):
            _lib.check(lib.gnr_upsample_int8_fwd(C.byref(self.p), C.byref(self.w), C.byref(self.s), C.c_void_p(self.img.data_ptr()),
                                                 C.c_void_p(self.ws.data_ptr()), self.ws.numel(), _stream_ptr(self.dev)), lib)
        return self.img


def neural_render_int8(x, params: Dict[str, torch.Tensor], n_blocks: int = 3, min_feat: int = 32, final_actvn: bool = True,
                       weights: Optional[Int8Weights] = None, cache=None, slots=None):
    """``neural_render`` in 8 bits: x [B, feat_nc, S, S] -- or x None with a ``FeatureMapCache`` and int64 ``slots`` [B] on its device --
    -> image [B, 3, S*2^n, S*2^n].  ``weights`` keeps the quantised weights from call to call; a call that is being captured quantises them
    in the graph instead, so that a replay follows its parameters.  Inference only."""
    int8._no_grad("neural_render_int8", x, getattr(cache, "scale", None), *params.values())
    dev = x if x is not None else getattr(cache, "q", None)
    if weights is None or (getattr(dev, "is_cuda", False) and torch.cuda.is_current_stream_capturing()):
        weights = Int8Weights()
    return _Call(params, weights, int(n_blocks), int(min_feat), bool(final_actvn), x, cache, slots)()


class GraphedUpsample8:
    """``neural_render_int8`` replayed from a HIP graph, one per input shape (or cache), device and parameter storage: the call is
    some thirty launches of a few microseconds.  The graph reads the quantised weights of ``weights``, refreshed before each replay if a
    parameter changed, and the biases and RGB weights in place; the input (a map, or the slots) is copied into the graph's own buffer.
    For one HIP stream, from any number of threads: between a call's copy into that buffer and its copy out of the image nobody else's
    work is enqueued.  Where there are more shapes and caches in use than ``max_entries``, the others run without a graph."""

    def __init__(self, weights: Int8Weights, max_entries: int = 4):
        self.weights, self.max_entries = weights, max_entries
        self.lock = threading.Lock()
        self.entries = RecentlyUsed(max_entries)
        self.captures = self.replays = 0

    def clear(self):
        with self.lock:
            self.entries.clear()

    def __call__(self, params, n_blocks, min_feat, final_actvn, x=None, cache=None, slots=None):
        int8._no_grad("neural_render_int8", x, getattr(cache, "scale", None), *params.values())
        with self.lock, self.weights.lock:
            return self._replay(params, n_blocks, min_feat, final_actvn, x, cache, slots)

    def _replay(self, params, n_blocks, min_feat, final_actvn, x, cache, slots):
        self.weights.refresh(params, n_blocks)
        given = x if x is not None else slots
        key = (tuple(given.shape), given.dtype, given.device, n_blocks, min_feat, bool(final_actvn)) + tuple(
            params[n].data_ptr() for n in renderer_param_names(n_blocks)) + tuple(r.q.data_ptr() for r in self.weights.rows.values())
        if cache is not None:
            key += (cache.q.data_ptr(), cache.scale.data_ptr(), tuple(cache.q.shape), cache.q.stride(), cache.scale.stride())
        ent = self.entries.get(key)
        if ent is None:
            if not self.entries.room():
                return _Call(params, self.weights, n_blocks, min_feat, final_actvn, x, cache, slots)()
            with torch.inference_mode(False), torch.no_grad():       # the static buffers outlive this call
                ent = self._capture(params, n_blocks, min_feat, final_actvn, x, cache, slots)
            self.entries.put(key, ent)
        graph, static, call = ent
        static.copy_(given)
        graph.replay()
        self.replays += 1
        return call.img.clone()

    def _capture(self, params, n_blocks, min_feat, final_actvn, x, cache, slots):
        given = x if x is not None else slots
        static = torch.empty(given.shape, dtype=given.dtype, device=given.device)
        static.copy_(given)
        call = _Call(params, self.weights, n_blocks, min_feat, final_actvn, static if x is not None else None, cache, static if x is None else None)
        if x is None and call.q.data_ptr() != cache.q.data_ptr():
            raise ValueError("GraphedUpsample8: the cache's rows are not on 16-byte boundaries; the graph would read a temporary copy")
        for n, t in call.params.items():
            if t.data_ptr() != params[n].data_ptr():
                raise ValueError("GraphedUpsample8: parameter %s is not contiguous; the graph would read a temporary copy" % n)
        if x is None and call.scale.data_ptr() != cache.scale.data_ptr():
            raise ValueError("GraphedUpsample8: the cache's scales are not contiguous; the graph would read a temporary copy")
        graph = capture_graph(given.device, call)
        if x is None:
            call.q = call.scale = None       # the caller's: the key holds their addresses, so a replay's caller has them, and a dropped cache is free
        self.captures += 1
        return graph, static, call


class Int8Renderers:
    """A ``GraphedUpsample8`` (with its ``Int8Weights``) per HIP stream: what two streams run at once shares no buffer.  Where there are more
    streams in use than ``max_streams``, the others get None: they run without a graph and quantise the weights in every call.  A copy
    starts empty: graphs and structs of device pointers are not copied."""

    def __init__(self, max_streams: int = 4):
        self.max_streams = max_streams
        self.streams = RecentlyUsed(max_streams)
        self.lock = threading.Lock()

    def __call__(self, dev) -> Optional[GraphedUpsample8]:
        key = (dev, torch.cuda.current_stream(dev).cuda_stream if dev.type == "cuda" else None)
        with self.lock:
            r = self.streams.get(key)
            if r is None and self.streams.room():
                r = GraphedUpsample8(Int8Weights())
                self.streams.put(key, r)
        return r

    def look_again(self):
        """The next call on each stream quantises its weights again."""
        with self.lock:
            for r in self.streams.values.values():
                with r.weights.lock:
                    r.weights.seen = None

    def clear(self):
        with self.lock:
            self.streams.clear()

    def __deepcopy__(self, memo):
        return Int8Renderers(self.max_streams)

    def __getstate__(self):
        return {"max_streams": self.max_streams}

    def __setstate__(self, state):
        self.__init__(state["max_streams"])
