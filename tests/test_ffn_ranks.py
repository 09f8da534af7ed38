"""The Llama model with the fused feed-forward block, planned over several (gloo) ranks, against the same model on one."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
from conftest import free_port


def _worker(rank, ws, shape, checkpoint, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(ws))
    dist.init_process_group("gloo", rank=rank, world_size=ws)
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor.placement_types import Replicate, Shard

    from autoparallel_b200 import AutoParallel, ForwardInputs
    from autoparallel_b200.models.llama3 import Transformer, llama3_debug

    mesh = init_device_mesh("cpu", shape, mesh_dim_names=("dp", "tp")[: len(shape)])
    cfg = llama3_debug(fused_ffn=True, fused_norm=True, ffn_checkpoint=checkpoint)
    B, S = 8, 64
    with torch.device("meta"):
        m = Transformer(cfg)

    def input_fn():
        return ForwardInputs((torch.randint(0, cfg.vocab_size, (B, S)),), {"labels": torch.randint(0, cfg.vocab_size, (B, S))})

    with AutoParallel(m, input_fn, mesh) as ap:
        ap.add_parameter_memory_constraint()
        ap.add_input_constraints([(Shard(0),) + (Replicate(),) * (mesh.ndim - 1)] * 2)
        ap.optimize_placement()
        pm = ap.apply_placement(executor="graph")
    pm.to_empty(device="cpu")
    pm.init_weights(seed=0)
    torch.manual_seed(1)
    tok, lab = (torch.randint(0, cfg.vocab_size, (B, S)) for _ in range(2))
    r0 = mesh.get_local_rank(0)
    loss = pm(tok.chunk(shape[0], 0)[r0], labels=lab.chunk(shape[0], 0)[r0])
    loss.backward()
    ref = Transformer(cfg)
    ref.init_weights(seed=0)
    rl = ref(tok, lab)
    rl.backward()
    worst = 0.0
    for p, p2 in zip(pm.parameters(), ref.parameters()):
        worst = max(worst, ((p.grad.full_tensor().float() - p2.grad).abs().max() / (p2.grad.abs().max() + 1e-12)).item())
    with torch.no_grad():
        inf = pm(tok.chunk(shape[0], 0)[r0], labels=lab.chunk(shape[0], 0)[r0])
    if rank == 0:
        q.put((loss.item(), rl.item(), worst, inf.item()))
    dist.destroy_process_group()


@pytest.mark.parametrize("shape,checkpoint", [((2,), "full"), ((2, 2), "full"), ((2,), "mx8")])
def test_ranks_match_one(shape, checkpoint):
    ws = 1
    for s in shape:
        ws *= s
    q = mp.get_context("spawn").SimpleQueue()
    mp.spawn(_worker, args=(ws, shape, checkpoint, free_port(), q), nprocs=ws, join=True)
    loss, ref, worst, inf = q.get()
    # (sums in another order may round a code the other way, a 64th of a block's largest value, in few of many terms)
    assert abs(loss - ref) < 1e-5 and abs(inf - ref) < 1e-5 and worst < (1e-4 if checkpoint == "full" else 1e-2)
