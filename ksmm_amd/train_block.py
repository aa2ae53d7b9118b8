"""Train gated Kronecker-sparse feed-forward blocks, then answer with them row by row:

    python -m ksmm_amd.train_block --gated 1,768,192,2 --down 1,192,768,2 6,64,64,1 --blocks 2 --rows 6272 --steps 40

Blocks of ``KSFeedForward`` (gated products, residual norms) learn what other random blocks of the same patterns answer to
random rows.  ``KSMuon`` updates the factors, SGD with momentum the norms' weights and gates.  A single row runs as a
captured graph, whose results are compared with the eager ones.  One JSON line: losses (of the targets' variance, before
and after), time of a training step, time of a row."""
import argparse
import json
import time

import torch
from torch import nn

from .block import KSFeedForward
from .muon import KSMuon


class KSStack(nn.Module):
    """Feed-forward blocks on one residual stream; the last block's norm leaves the answer."""

    def __init__(self, gated, down, blocks, **how):
        super().__init__()
        self.blocks = nn.ModuleList(KSFeedForward(gated, down, **how) for _ in range(blocks))

    def forward(self, residual):
        normed = self.blocks[0].begin(residual)
        for block in self.blocks:
            normed, residual = block(normed, residual)
        return normed


@torch.enable_grad()
def train(model, batches, steps, lr=0.02, lr_norm=0.02, scale=1024.0):
    """``steps`` steps over (input, target) pairs; the loss of each, of the target's variance, on the device.  Gradients
    are scaled by ``scale`` for fp16's sake: orthogonalised updates do not depend on it, the others divide by it."""
    muon = KSMuon(model, lr=lr)
    rest = KSMuon.others(model)
    sgd = torch.optim.SGD(rest, lr=lr_norm / scale, momentum=0.9)
    losses = []
    for i in range(steps):
        x, target = batches[i % len(batches)]
        for opt in (muon, sgd):
            opt.zero_grad(set_to_none=True)
        off = (model(x) - target).float()
        loss = (off * off).mean() / target.float().var()
        (loss * (scale * target.shape[1 if not model.blocks[0].norm.bs_last else 0])).backward()
        muon.step()
        sgd.step()
        losses.append(loss.detach())
    return losses


class OneRow:
    """Answers of a trained stack to single rows: the launches are captured once and replayed."""

    def __init__(self, model, features, dtype):
        self.model = model
        self.x = torch.zeros((features, 1) if model.blocks[0].norm.bs_last else (1, features), dtype=dtype, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), torch.no_grad():
            model(self.x)  # (workspaces are made outside the capture)
        torch.cuda.current_stream().wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph), torch.no_grad():
            self.y = model(self.x)

    def __call__(self, row):
        self.x.copy_(row)
        self.graph.replay()
        return self.y.clone()


def pattern(text):
    return tuple(int(v) for v in text.split(","))


def main(argv=None):
    ap = argparse.ArgumentParser(prog="python -m ksmm_amd.train_block", description=__doc__.split("\n")[0])
    ap.add_argument("--gated", type=pattern, default=(1, 768, 192, 2), help="a,b,c,d of both products of the gated projection")
    ap.add_argument("--down", type=pattern, nargs="+", default=[(1, 192, 768, 2), (6, 64, 64, 1)], help="factors behind it, in the order they are applied")
    ap.add_argument("--blocks", type=int, default=2)
    ap.add_argument("--rows", type=int, default=6272, help="rows of a training batch")
    ap.add_argument("--batches", type=int, default=8)
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--dtype", choices=("fp16", "fp32"), default="fp16")
    ap.add_argument("--bs-last", type=int, choices=(0, 1), default=0)
    ap.add_argument("--seed", type=int, default=0)
    args = ap.parse_args(argv)
    if args.steps < 1 or args.rows < 1 or args.blocks < 1 or args.batches < 1:
        ap.error("steps, rows, blocks and batches are at least 1")
    torch.manual_seed(args.seed)
    dtype = {"fp16": torch.float16, "fp32": torch.float32}[args.dtype]
    how = dict(dtype=dtype, bs_last=bool(args.bs_last), device="cuda")
    teacher, model = KSStack(args.gated, args.down, args.blocks, **how), KSStack(args.gated, args.down, args.blocks, **how)
    features = model.blocks[0].gated.in_size
    with torch.no_grad():
        batches = []
        for _ in range(args.batches):
            x = torch.randn((features, args.rows) if args.bs_last else (args.rows, features), device="cuda").to(dtype)
            batches.append((x, teacher(x)))
    train(KSStack(args.gated, args.down, args.blocks, **how), batches, 1)  # (what the first call of each kernel sets up)
    torch.cuda.synchronize()
    start = time.perf_counter()
    losses = train(model, batches, args.steps)
    torch.cuda.synchronize()
    step_ms = (time.perf_counter() - start) / args.steps * 1e3

    one = OneRow(model, features, dtype)
    worst = 0.0
    x, _ = batches[0]
    for i in range(min(8, args.rows)):
        row = x[:, i:i + 1].contiguous() if args.bs_last else x[i:i + 1].contiguous()
        with torch.no_grad():
            eager = model(row)
        worst = max(worst, float((one(row) - eager).abs().max()))
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for _ in range(200):
        one.graph.replay()
    end.record()
    torch.cuda.synchronize()
    result = {"gated": args.gated, "down": args.down, "blocks": args.blocks, "rows": args.rows, "steps": args.steps, "dtype": args.dtype,
              "bs_last": args.bs_last, "data": "synthetic", "first_loss": float(losses[0]), "last_loss": float(losses[-1]),
              "ms_per_step": step_ms, "us_per_row": begin.elapsed_time(end) / 200 * 1e3, "graph_minus_eager": worst}
    print(json.dumps(result), flush=True)
    return result


if __name__ == "__main__":
    main()
