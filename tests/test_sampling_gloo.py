"""Sampling and top logits under tensor parallelism: two gloo ranks draw what one rank draws (the ranks' own generators differ:
rank 0's numbers count), and give its top logits, with the batch in two pieces, in one, and token by token."""
import os
import random

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from test_large_model import _continuous_case, _oracle_cell
from xlstm_b200.large_model import ContinuousDecoder, LargeConfig, LargeModel, Sampling, procedural_state_dict

CFG = LargeConfig(embedding_dim=128, num_heads=2, num_blocks=2, vocab_size=64)
PER_ROW = dict(temperature=torch.tensor([0.9, 1.3, 0.0, 0.7]), top_k=torch.tensor([0, 12, 0, 5]), top_p=0.95, min_p=torch.tensor([0.0, 0.02, 0.0, 0.0]))


def _rows(n):
    return Sampling(*(v[:n] if torch.is_tensor(v) else v for v in PER_ROW.values()))


def _everything(model, seed):
    """Tokens of batches of 4 (two pieces), 3 (one piece) and 1, of a decoder's slots, and the top logits of two batches."""
    g = torch.Generator().manual_seed(1)
    out = []
    for B, S in ((4, 18), (3, 16), (1, 7)):
        prompt = torch.randint(0, 64, (B, S), generator=g)
        out.append(model.generate(prompt, 6, sampling=_rows(B), generator=torch.Generator().manual_seed(seed))[0])
        if B > 1:
            out += model.top_logits(prompt, 5, 2.0)
    prompts, counts = _continuous_case()
    settings = [Sampling(0.8, 20, 0.9), Sampling(), Sampling(0.0), Sampling(1.2, 0, 1.0, 0.05), Sampling(1.0, 5), Sampling(0.7, 0, 0.8), Sampling(1.5, 1)]
    out += ContinuousDecoder(model, 3, sampling=True).run(prompts, counts, sampling=settings, generator=torch.Generator().manual_seed(seed))
    return out


def _worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.set_num_threads(2)
    model = LargeModel(CFG, procedural_state_dict(CFG, 4), "cpu", torch.float32, tp_rank=rank, tp_world=world, cell_ops=_oracle_cell())
    out = _everything(model, 5 + rank)
    gathered = [None] * world
    dist.all_gather_object(gathered, [t.tolist() for t in out])
    if rank == 0:
        q.put(gathered)
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_draw_the_tokens_of_one():
    want = _everything(LargeModel(CFG, procedural_state_dict(CFG, 4), "cpu", torch.float32, cell_ops=_oracle_cell()), 5)
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = 33000 + random.randint(0, 2000)
    procs = [ctx.Process(target=_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    gathered = q.get(timeout=300)
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    assert gathered[0] == gathered[1]
    for a, b in zip(gathered[0], want):
        if b.is_floating_point():   # (the ranks' partial sums are added in another order)
            torch.testing.assert_close(torch.tensor(a), b, rtol=1e-4, atol=1e-4)
        else:
            assert a == b.tolist()
