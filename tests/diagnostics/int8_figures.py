"""GPU: the figures that stand beside the 8-bit operators.

    python tests/diagnostics/int8_figures.py times          the renderer through its HIP graphs, 8-bit (from maps, from cached rows) and fp32,
                                                            and how far the 8-bit image is from the fp32 one
    rocprofv3 --kernel-trace --output-format csv -d DIR -o NAME -- python3 tests/diagnostics/int8_figures.py run cases|renderer|same
                                                            calls for a profiler: the cases of perf/operators.py (three sets of inputs in turn), the
                                                            renderer without graphs, or maps that are read again and again
    python tests/diagnostics/int8_figures.py table DIR/NAME_kernel_trace.csv [DIR/NAME_counter_collection.csv]
                                                            the table of such a run (a --pmc WRITE_SIZE run gives the second file)
-> profiles/int8_operators_kernels.txt, profiles/int8_renderer.txt"""
import collections
import csv
import math
import os
import re
import statistics
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, ROOT)


def renderer(precision):
    import torch
    import gazenerf_amd as G
    from gazenerf_amd import synth
    net = G.NeuralRendererAMD(precision=precision)
    net.load_state_dict(dict(net.state_dict(), **{k: v.reshape(net.state_dict()[k].shape) for k, v in synth.hash_renderer_params(seed=2).items()}))
    return net.to("cuda").eval()


def maps(B):
    from gazenerf_amd import synth
    return synth.synth_featmap(B, 258, 64, seed=4).to("cuda")


def times():
    import torch
    import gazenerf_amd as G
    from gazenerf_amd import _lib
    print("build: %s" % _lib.build_info())
    nets = {p: renderer(p) for p in ("int8", "fp32")}
    cache = G.FeatureMapCache(8)

    def us(call, n=40):
        for _ in range(5):
            call()
        out = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(n):
                call()
            b.record()
            torch.cuda.synchronize()
            out.append(a.elapsed_time(b) * 1e3 / n)
        return statistics.median(out)

    with torch.no_grad():
        for B in (1, 2, 7):
            x, slots = maps(B), torch.arange(B, device="cuda")
            cache.write(slots, x)
            sides = (lambda: nets["int8"](x), lambda: nets["int8"].render_cached(cache, slots), lambda: nets["fp32"](x))
            print("B = %d: 8-bit %.0f us, from cached rows %.0f, fp32 %.0f" % ((B,) + tuple(us(s) for s in sides)))
        a, b = nets["int8"](x).double(), nets["fp32"](x).double()
        print("8-bit against fp32 image, 7 maps: rms %.2e, largest %.2e, %.1f dB (a value of 1 is 0 dB); the fp32 image's own spread: standard deviation %.3f" % (
            float((a - b).pow(2).mean().sqrt()), float((a - b).abs().max()), -10 * math.log10(float((a - b).pow(2).mean())), float(b.std())))


def run(what):
    import torch
    import gazenerf_amd as G
    with torch.no_grad():
        if what == "cases":
            sys.path.insert(0, os.path.join(ROOT, "perf"))
            import operators
            operators.own = True
            for case in operators.listed():
                states = [operators.prepare(case, s) for s in range(3)]
                for i in range(15):
                    operators.run(states[i % 3])
                torch.cuda.synchronize()
        elif what == "renderer":
            from gazenerf_amd.upsample8 import Int8Weights
            net, weights = renderer("int8"), Int8Weights()
            params = {k: v for k, v in net.named_parameters() if k != "bg_featmap"}
            for B in (1, 7):
                x = maps(B)
                for _ in range(15):
                    G.neural_render_int8(x, params, weights=weights)
                torch.cuda.synchronize()
        else:
            cache, x, slots = G.FeatureMapCache(64), maps(8).repeat(8, 1, 1, 1), torch.arange(64, device="cuda")
            cache.write(slots, x)
            for _ in range(15):
                cache.read(slots)
            for _ in range(15):
                cache.write(slots, x)
    torch.cuda.synchronize()
    print("done", flush=True)


def table(trace, counters=None):
    names = {}

    def name(n):
        if n not in names:
            m = n.split(".kd")[0]
            if m.startswith("_Z"):
                m = subprocess.run(["c++filt"], input=m.replace("DF16b", "u6__bf16").replace("DF16_", "Dh"), capture_output=True, text=True).stdout.strip()
            m = re.sub(r"bool _Accum, bool, E", "__bf16, true", m).replace("void ", "").replace("gnr::", "").replace("half", "_Float16")
            names[n] = re.sub(r"\(.*", "", m)
        return names[n]

    rows = collections.OrderedDict()
    for r in sorted(csv.DictReader(open(trace)), key=lambda r: int(r["Start_Timestamp"])):
        if "gnr" in r["Kernel_Name"]:
            threads = int(r["Grid_Size_X"]) * int(r["Grid_Size_Y"])
            rows.setdefault((name(r["Kernel_Name"]), threads, r["Workgroup_Size_X"]), []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
    writes = {}
    if counters:
        for r in csv.DictReader(open(counters)):
            if "gnr" in r["Kernel_Name"] and r["Counter_Name"] == "WRITE_SIZE":
                writes.setdefault((name(r["Kernel_Name"]), int(r["Grid_Size"]), r["Workgroup_Size"]), []).append(float(r["Counter_Value"]))
    print("%-60s %10s x %4s %4s %9s %9s %9s" % ("kernel", "threads", "block", "n", "median us", "min us", "MB written"))
    for k, us in rows.items():
        w = statistics.median(writes[k]) * 1.024e-3 if k in writes else float("nan")
        print("%-60s %10d x %4s %4d %9.2f %9.2f %9.2f" % (k[0][:60], k[1], k[2], len(us), statistics.median(us), min(us), w))


if __name__ == "__main__":
    {"times": lambda: times(), "run": lambda: run(sys.argv[2]), "table": lambda: table(*sys.argv[2:])}[sys.argv[1]]()
