"""A routed FFN with MXFP4 experts: y = x + sum_j w_j E_ids[j](x).

The router's logits (f32, `gemv`, or `gemm_tf32x3w` for many rows) go through the grouped route, and
each row's experts through the routed MXFP4 products with the GELU gate
between them; the ranks are combined onto the row. `RoutedExperts` keeps
the experts' tables at 17 bits to four weights, quantised on the device
from f32, and launches the block for any number of rows up to `rows` on its
context's stream, so that a decode step and a prompt take the same calls,
alone or captured in a graph:

    experts = RoutedExperts(ctx, router, gate_up, down, top_k=8, rows=512)
    experts.launch(x, y, m)

`python -m furykernel_b200.experts` times the block at a few row counts.
"""

import argparse

import numpy as np

from furykernel_b200 import _native as N


# Rows past which the router is a tensor-core GEMM (the block with 64 experts,
# 2048 x 1408: 32 rows 188 us by gemv and 199 by GEMM, 64 rows 200 and 186, 511
# rows 1032 and 318).
GEMM_ROWS = 48


class Mxfp4Table:
    """Weights [entries, n, kk] as codes [entries, n, kk / 2] and a scale a
    block of 32 [entries, n, kk / 32], from f32 in the host's or the
    device's memory."""

    def __init__(self, ctx: N.Context, weights, entries: int, n: int, kk: int):
        self.entries, self.n, self.kk = entries, n, kk
        if weights.size != entries * n * kk if isinstance(weights, np.ndarray) else weights.nbytes != 4 * entries * n * kk:
            raise N.Refused(N.FKC_ERR_ARGUMENT, f"MXFP4 table: the weights are not {entries} x {n} x {kk}.")
        whole = ctx.to_device(weights.astype(np.float32)) if isinstance(weights, np.ndarray) else weights
        self.codes = ctx.empty((entries, n, kk // 2), np.uint8)
        self.scales = ctx.empty((entries, n, kk // 32), np.uint8)
        ctx.launch("quant_mxfp4", {"rows": entries * n, "k": kk, "ldx": kk}, [whole, self.codes, self.scales])
        if whole is not weights:
            ctx.sync()
            whole.free()

    def free(self) -> None:
        self.codes.free()
        self.scales.free()


class RoutedExperts:
    """router [E, d], gate_up [E, 2 ffn, d] (each expert's gate rows, then its
    up rows), down [E, d, ffn]; `bias` [E] is added to the scores that pick,
    not to the weights."""

    def __init__(self, ctx: N.Context, router: np.ndarray, gate_up, down, ffn: int, top_k: int, rows: int,
                 groups: int = 1, top_groups: int = 1, group_by: int = 1, sigmoid: bool = False,
                 renorm: bool = True, factor: float = 1.0, bias: np.ndarray = None):
        e, d = router.shape
        if bias is not None and bias.size != e:
            raise N.Refused(N.FKC_ERR_ARGUMENT, f"routed experts: the bias has {bias.size} values, not {e}.")
        self.ctx, self.e, self.d, self.ffn, self.k, self.rows = ctx, e, d, ffn, top_k, rows
        self.route = {"n": e, "k": top_k, "groups": groups, "top_groups": top_groups, "group_by": group_by,
                      "sigmoid": int(sigmoid), "renorm": int(renorm), "ldx": e, "factor": factor}
        self.router = ctx.to_device(router.astype(np.float32))
        self.bias = None if bias is None else ctx.to_device(bias.astype(np.float32))
        self.gate_up = Mxfp4Table(ctx, gate_up, e, 2 * ffn, d)
        self.down = Mxfp4Table(ctx, down, e, d, ffn)
        self.parts = ctx.empty((2, rows, d)) if rows > GEMM_ROWS else None  # the rows as TF32 parts
        self.logits, self.ids = ctx.zeros((rows, e)), ctx.zeros((rows, top_k), np.uint32)
        self.ws, self.gu = ctx.zeros((rows, top_k)), ctx.zeros((rows, top_k * 2 * ffn))
        self.act, self.out = ctx.zeros((rows, top_k * ffn)), ctx.zeros((rows, top_k * d))
        # One workspace: the products run one after the other.
        self.work = ctx.alloc(max(N.linear_mxfp4_work(2 * ffn, d, rows, e, top_k),
                                  N.linear_mxfp4_work(d, ffn, rows, e, top_k)), np.uint8)

    def _product(self, t: Mxfp4Table, x, y, m: int, per_rank: bool) -> None:
        self.ctx.launch("linear_routed_mxfp4",
                        {"entries": self.e, "n": t.n, "kk": t.kk, "m": m, "k": self.k,
                         "ldx": t.kk * (self.k if per_rank else 1), "ldy": self.k * t.n, "per_rank": int(per_rank)},
                        [t.codes, t.scales, self.ids, x, y, self.work])

    def launch(self, x, y, m: int) -> None:
        """y [m, d] = x [m, d] + the weighted sum of each row's experts."""
        if not 0 < m <= self.rows:
            raise N.Refused(N.FKC_ERR_ARGUMENT, f"routed experts: {m} rows, outside 1..{self.rows}.")
        for name, b in (("x", x), ("y", y)):
            if isinstance(b, N.DeviceBuffer) and b.nbytes < 4 * m * self.d:
                raise N.Refused(N.FKC_ERR_ARGUMENT, f"routed experts: {name} holds fewer than {m} rows of {self.d}.")
        if m > GEMM_ROWS:
            self.ctx.launch("gemm_tf32x3w", {"M": m, "N": self.e, "K": self.d, "ldc": self.e},
                            [x, self.parts, self.parts.at(self.rows * self.d), self.router, self.logits])
        else:
            self.ctx.launch("gemv", {"n": self.e, "k": self.d, "m": m, "split": 1, "ldx": self.d, "ldy": self.e},
                            [self.router, x, self.logits])
        bias = [] if self.bias is None else [self.bias]
        self.ctx.launch("route_grouped_bias" if bias else "route_grouped", {**self.route, "m": m},
                        [self.logits, *bias, self.ids, self.ws])
        self._product(self.gate_up, x, self.gu, m, False)
        self.ctx.launch("gated_gelu", {"segments": m * self.k, "f": self.ffn}, [self.gu, self.act])
        self._product(self.down, self.act, self.out, m, True)
        self.ctx.launch("combine_ranks_add", {"m": m, "k": self.k, "d": self.d}, [x, self.ws, self.out, y])

    def free(self) -> None:
        for b in (self.router, self.bias, self.parts, self.gate_up, self.down, self.logits, self.ids, self.ws, self.gu, self.act,
                  self.out, self.work):
            if b is not None:
                b.free()


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--experts", type=int, default=64)
    p.add_argument("--top-k", type=int, default=8)
    p.add_argument("--d", type=int, default=2048)
    p.add_argument("--ffn", type=int, default=1408)
    p.add_argument("--groups", type=int, default=8)
    p.add_argument("--top-groups", type=int, default=4)
    p.add_argument("--rows", type=int, nargs="+", default=[1, 8, 64, 511, 2048])
    a = p.parse_args()
    rng = np.random.default_rng(512)
    with N.Context(0) as ctx:
        gate_up, down = ctx.empty((a.experts, 2 * a.ffn, a.d)), ctx.empty((a.experts, a.d, a.ffn))
        ctx.fill_normal(gate_up, 1, 0.0, 0.02)
        ctx.fill_normal(down, 2, 0.0, 0.02)
        block = RoutedExperts(ctx, rng.normal(0, 0.02, (a.experts, a.d)), gate_up, down, a.ffn, a.top_k, max(a.rows),
                              groups=a.groups, top_groups=a.top_groups, group_by=2, sigmoid=True,
                              bias=rng.normal(0, 0.1, a.experts))
        gate_up.free()
        down.free()
        x = ctx.to_device(rng.normal(0, 1, (max(a.rows), a.d)).astype(np.float32))
        y = ctx.zeros((max(a.rows), a.d))
        for m in a.rows:
            ctx.capture_begin()
            block.launch(x, y, m)
            g = ctx.capture_end()
            ms = g.time(3, 20) / 20
            g.destroy()
            chosen = len(np.unique(block.ids.download()[:m]))
            read = chosen * 3 * a.d * a.ffn * 17 / 32
            print(f"{m} rows, {chosen} experts: {ms * 1e3:.1f} us, {read / ms * 1e-6:.0f} GB/s of weights, "
                  f"{6 * m * a.top_k * a.d * a.ffn / ms * 1e-9:.1f} TFLOP/s")
        if ctx.status():
            raise SystemExit("a wait ran out")
        block.free()


if __name__ == "__main__":
    main()
