"""Sampling and the divergence of a column-sharded lm_head: the gathered row is the whole row, and every rank
draws the same token (world_size-2 gloo ranks on the CPU, plain forms in place of the kernels)."""

import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import _logits as R
from mlxturbo_b200 import distributed as D


def _port() -> int:
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _weights():
    g = torch.Generator().manual_seed(0)
    V, K = 64, 32
    return torch.randn((V, K), generator=g), torch.zeros((V, 1)), torch.zeros((V, 1)), torch.randn((3, 2, K), generator=g)


def _matmul(x, w, s, b, group_size, bits):
    return x @ w.T


def _sampler(logits, u, temperature=1.0, top_k=0):
    rows = logits.reshape(-1, logits.shape[-1])
    ids = [R.sample(row, v, temperature, top_k) for row, v in zip(rows, u.reshape(-1))]
    return torch.tensor(ids).reshape(u.shape)


def _loss(logits, tv, ti, temperature=1.0):
    rows = logits.reshape(-1, logits.shape[-1])
    out = [R.distill(r, a, b, temperature)[0] for r, a, b in zip(rows, tv.flatten(0, -2), ti.flatten(0, -2))]
    return torch.tensor(out).reshape(tv.shape[:-1])


def _calls(head, x):
    u = torch.linspace(0.05, 0.95, 6).reshape(3, 2)
    tv, ti = (x @ _weights()[0].T + 0.1).topk(4, dim=-1)
    return (head.sample(x, u, sampler=_sampler, temperature=0.7, top_k=9),
            head.distill_loss(x, tv, ti, loss=_loss, temperature=2.0), head.topk(x, 4))


def _rank(rank, world, port, queue):
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)
    w, s, b, x = _weights()
    head = D.ColumnShardedLMHead.from_full(w, s, b, matmul=_matmul)
    assert head.shard_rows == 32
    ids, loss, (values, top) = _calls(head, x)
    queue.put((rank, ids.tolist(), loss.tolist(), top.tolist()))
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_draw_what_one_draws():
    w, s, b, x = _weights()
    ids, loss, (values, top) = _calls(D.ColumnShardedLMHead.from_full(w, s, b, matmul=_matmul), x)
    assert ids.shape == loss.shape == (3, 2)
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    port = _port()
    ranks = [ctx.Process(target=_rank, args=(r, 2, port, queue)) for r in range(2)]
    for p in ranks:
        p.start()
    got = [queue.get(timeout=120) for _ in ranks]
    for p in ranks:
        p.join(60)
        assert p.exitcode == 0
    for _, i, lo, t in got:
        assert i == ids.tolist() and t == top.tolist()
        torch.testing.assert_close(torch.tensor(lo), loss, rtol=1e-5, atol=0)


@pytest.mark.gpu
def test_one_gpu():
    from mlxturbo_b200 import ops

    g = torch.Generator().manual_seed(1)
    w, s, b = ops.quantize((torch.randn((4096, 256), generator=g) * 0.2).cuda(), dtype=torch.bfloat16)
    x = torch.randn((5, 256), generator=g).bfloat16().cuda()
    head = D.ColumnShardedLMHead.from_full(w, s, b, group_size=64, bits=4)
    logits = ops.quantized_matmul(x, w, s, b)
    u = torch.rand(5, generator=g).cuda()
    assert torch.equal(head.sample(x, u, temperature=0.8, top_p=0.9), ops.sample(logits, u, temperature=0.8, top_p=0.9))
    values, ids = head.topk(x, 7)
    v, i = ops.topk(logits, 7)
    assert torch.equal(ids, i) and torch.equal(values, v.float()) and values.dtype == torch.float32
    assert torch.equal(head.sample(x, u, temperature=0), head.argmax(x))
    tv, ti, lse = ops.topk(logits + 0.1 * torch.randn_like(logits), 16, logsumexp=True)
    assert torch.equal(head.distill_loss(x, tv, ti, teacher_logsumexp=lse),
                       ops.distill_loss(logits, tv, ti, teacher_logsumexp=lse))
