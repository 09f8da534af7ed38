"""A mixture-of-experts layer with grouped sigmoid routing and 4-bit experts (MXFP4): planned for 8 fake ranks, trained for some steps on one device, and
then served with weights that are held in 4 bits.

    python examples/example_moe_mx4.py [--steps 20]

The routed block is ``moe_route`` (scores, a balance bias for the choice, groups, top-k, renormalised weights), the capacity dispatch, ``mx4_matmul`` for the
experts' projections, and the weighted combine.  ``router_bias`` is moved after every step towards the experts that got too few tokens."""
import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch
from torch.distributed.tensor.placement_types import Shard

import autoparallel_b200.ops as K
from autoparallel_b200 import AutoParallel, ForwardInputs
from autoparallel_b200.models.moe import MoEFFN, MoETransformer, moe_debug
from examples._fake import fake_mesh


def config(**kw):
    return moe_debug(expert_mode="planner", expert_format="mx4", router_score="sigmoid", router_groups=4, router_top_groups=2, router_scale=2.5,
                     num_experts=16, top_k=4, dispatch_blocks=8, max_seq_len=64, **kw)


def plan():
    cfg, mesh = config(), fake_mesh((8,), ("dp",))
    with torch.device("meta"):
        model = MoETransformer(cfg)

    def input_fn():
        return ForwardInputs((torch.randint(0, cfg.vocab_size, (8, 64)),), {"labels": torch.randint(0, cfg.vocab_size, (8, 64))})

    with AutoParallel(model, input_fn, mesh, plan_device="B200") as ap:
        ap.add_parameter_memory_constraint()
        ap.add_input_constraints([(Shard(0),)] * 2)
        sol = ap.optimize_placement()
        seen = set()
        for n in ap.gm.graph.nodes:
            name = str(n.target).split(".")[1] if n.op == "call_function" and ("mx4_" in str(n.target) or "moe_route" in str(n.target)) else None
            if name and name not in seen:
                seen.add(name)
                outs = sol[n].output_specs
                outs = outs if isinstance(outs, (tuple, list)) else [outs]
                print(f"{name:14s} in {[str(tuple(i.placements)) for i in sol[n].input_specs]} -> {[tuple(o.placements) for o in outs]}")
        print("collectives:", ap.lower().num_collectives)


def train(device, steps):
    """One layer learns to reproduce a random linear map."""
    torch.manual_seed(0)
    cfg = config(dim=256, expert_hidden=128, shared_hidden=128, capacity_factor=2.0)
    dtype = torch.bfloat16 if device == "cuda" else torch.float32
    layer = MoEFFN(cfg).to(device)
    layer.init_weights(0.05)
    layer.to(dtype)
    layer.router_bias = layer.router_bias.float()
    target = torch.randn(cfg.dim, cfg.dim, device=device, dtype=dtype) * cfg.dim**-0.5
    opt = torch.optim.SGD(layer.parameters(), lr=1.0, momentum=0.9)
    for step in range(steps):
        x = torch.randn(4, 64, cfg.dim, device=device, dtype=dtype)
        loss = (layer(x) - x @ target).float().square().mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        with torch.no_grad():
            load = torch.bincount(layer.route(x)[1].flatten(), minlength=cfg.num_experts).float()
            layer.router_bias += 0.001 * torch.sign(load.mean() - load)
        if step % 5 == 0 or step == steps - 1:
            print(f"step {step:3d}  loss {loss.item():.4f}  load {int(load.min())} .. {int(load.max())}")
    return layer


@torch.no_grad()
def serve(layer):
    """The experts' up projections for a few tokens, from weights quantised once."""
    codes, scales = K.mx4_quantize(layer.w1.transpose(1, 2))  # [E, hidden, dim], blocks along dim
    held = codes.numel() + scales.numel()
    x = torch.randn(layer.cfg.num_experts, 2, layer.cfg.dim, device=layer.w1.device, dtype=layer.w1.dtype)
    y = K.mx4_linear(x, codes, scales)
    same = torch.equal(y, K.mx4_matmul(x, layer.w1, trans_b=False))
    print(f"served {tuple(x.shape)} -> {tuple(y.shape)} from {held} bytes ({layer.w1.numel() * layer.w1.element_size()} before); as in training: {same}")


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    plan()
    serve(train("cuda" if torch.cuda.is_available() else "cpu", a.steps))


if __name__ == "__main__":
    main()
