"""A decoder MLP with 4-bit weights: the MXFP4 operators as a program uses them.

    python examples/mxfp4_mlp.py [--rows 8] [--hidden 4096] [--inner 14336]

When the weights are loaded they are quantised (mxfp4_encode_rows) and packed (mxfp4_pack) once.  Every step then quantises the
activations of each projection - per row to E4M3 (fp8_encode_rows), or in blocks to MXFP4 (mxfp4_encode_rows) - and multiplies
(mxfp4_gemm_fp8act, mxfp4_gemm).  Prints how far the outputs are from the same MLP in bf16, how much of that is the weights'
quantisation alone (their values brought back by mxfp4_decode_rows), and the time of a step.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import rocm_dev_amd as sg  # noqa: E402


def empty(*shape, dtype=torch.uint8):
    return torch.empty(shape, dtype=dtype, device="cuda")


class Linear:
    """n x k weights in MXFP4, packed; `values` are what the codes stand for."""

    def __init__(self, W):
        self.n, self.k = W.shape
        Q, S = empty(self.n, self.k // 2), empty(self.n, self.k // 32)
        sg.mxfp4_encode_rows(W, Q, S, check=True)
        self.P = empty(sg.mxfp4_packed_bytes(self.n, self.k))
        sg.mxfp4_pack(Q, S, self.P, check=True)
        self.values = torch.empty_like(W)
        sg.mxfp4_decode_rows(Q, S, self.values, check=True)

    def __call__(self, X, activations):
        m = X.shape[0]
        D = empty(m, self.n, dtype=torch.bfloat16)
        if activations == "mxfp4":
            A, SA = empty(m, self.k // 2), empty(m, self.k // 32)
            sg.mxfp4_encode_rows(X, A, SA, check=True)
            sg.mxfp4_gemm(A, SA, self.P, D, check=True)
        else:
            A, row = empty(m, self.k), empty(m, dtype=torch.float32)
            sg.fp8_encode_rows(X, A, row, check=True)
            sg.mxfp4_gemm_fp8act(A, self.P, D, None, row, check=True)
        return D


def mlp(X, gate_up, down):
    gate, up = gate_up(X).float().chunk(2, 1)
    return down((torch.nn.functional.silu(gate) * up).bfloat16())


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--rows", type=int, default=8)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--inner", type=int, default=14336)
    args = ap.parse_args(argv)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(0)

    def weights(n, k):
        return (torch.randn((n, k), generator=gen, device="cuda") * k ** -0.5).bfloat16()

    W1, W2 = weights(2 * args.inner, args.hidden), weights(args.hidden, args.inner)
    X = torch.randn((args.rows, args.hidden), generator=gen, device="cuda").bfloat16()
    gate_up, down = Linear(W1), Linear(W2)

    def off(a, b):
        return ((a.float() - b.float()).norm() / b.float().norm()).item()

    want = mlp(X, lambda x: x @ W1.t(), lambda x: x @ W2.t())
    dequantised = mlp(X, lambda x: x @ gate_up.values.t(), lambda x: x @ down.values.t())
    print("4-bit weights, bf16 activations: %.3f off the bf16 MLP" % off(dequantised, want))
    result = {}
    for activations in ("e4m3", "mxfp4"):
        def step():
            return mlp(X, lambda x: gate_up(x, activations), lambda x: down(x, activations))
        Y = step()
        torch.cuda.synchronize()
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(20):
            step()
        end.record()
        torch.cuda.synchronize()
        result[activations] = (off(Y, want), off(Y, dequantised))
        print("4-bit weights, %s activations: %.3f off the bf16 MLP, %.3f off bf16 activations; %.1f us a step"
              % (activations, *result[activations], begin.elapsed_time(end) / 20 * 1e3))
    return result


if __name__ == "__main__":
    main()
