"""One feed-forward layer of a mixture of experts on 4-bit weights, as a serving program runs it.

    python examples/moe_layer.py [--tokens 1 64 2048] [--experts 64] [--top 4] [--width 4096] [--inner 1536]

The weights are quantised once (MX4). A step routes each token to its experts, multiplies its row with their gate and up
weights (SiLU of the gate times up), and joins the second products by the router's weights. Each step's result is compared
with the same layer computed in 64 bits from the dequantised weights, and timed."""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.realpath(__file__)), os.pardir, "gen9-gpu-blas_amd"))
import gen9blas  # noqa: E402


def layer(x, router, up, gate, down, top):
    logits = gen9blas.gemm(x, router)                                   # tokens × experts
    ids, weights = gen9blas.moe_route(logits, top)
    inner = gen9blas.moe_gemm(x, ids, up, gate=gate)                    # tokens × top × inner
    return ids, weights, gen9blas.moe_gemm(inner, ids, down, weights=weights)


def exact(x, ids, weights, up, gate, down):
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for e in torch.unique(ids).tolist():
        t, s = torch.nonzero(ids == e, as_tuple=True)
        rows = x[t].double()
        z = rows @ gate[e].double().t()
        inner = z * torch.sigmoid(z) * (rows @ up[e].double().t())
        y.index_add_(0, t, weights[t, s, None].double() * (inner @ down[e].double().t()))
    return y


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--tokens", type=int, nargs="+", default=[1, 64, 2048])
    p.add_argument("--experts", type=int, default=64)
    p.add_argument("--top", type=int, default=4)
    p.add_argument("--width", type=int, default=4096)
    p.add_argument("--inner", type=int, default=1536)
    p.add_argument("--steps", type=int, default=50)
    a = p.parse_args()
    g = torch.Generator(device="cuda").manual_seed(0)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda") * scale

    up, gate = (gen9blas.mx4_quantize(normal(a.experts, a.inner, a.width, scale=a.width ** -0.5)) for _ in range(2))
    down = gen9blas.mx4_quantize(normal(a.experts, a.width, a.inner, scale=a.inner ** -0.5))
    router = normal(a.width, a.experts, scale=2 * a.width ** -0.5).half()
    gen9blas.set_nowait(True)   # everything is on the GPU: calls queue on the library's stream
    for tokens in a.tokens:
        x = normal(tokens, a.width).half()
        ids, weights, y = layer(x, router, up, gate, down, a.top)
        gen9blas.flush()
        ref = exact(x, ids, weights, *(gen9blas.mx4_dequantize(w) for w in (up, gate, down)))
        error = float((y.double() - ref).norm() / ref.norm())
        start = time.perf_counter()
        for _ in range(a.steps):
            layer(x, router, up, gate, down, a.top)
        gen9blas.flush()
        print(f"{tokens:5d} tokens, {a.top} of {a.experts} experts, {a.width} x {a.inner}: {(time.perf_counter() - start) / a.steps * 1e6:8.1f} us a layer, "
              f"relative error {error:.1e}")
        if not error < 2e-3:   # FP16 roundings of the inner values and the result, 2^-12 each
            sys.exit("the layer's result is wrong")


if __name__ == "__main__":
    main()
