"""Adapters and logits of a sharded decoder on CPU ranks over gloo: column- and row-split
adapters give the unsharded sums, the gathered logits are the whole rows on every rank."""

import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def _worker(rank, world, port):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    from qextract_infer_b200.tp_shard import gather_logits, shard_adapters, shard_vocab
    g = torch.Generator().manual_seed(3)
    n, K, r, N, b = 3, 32, 8, 48, 5
    A, B, x = torch.randn(n, K, r, generator=g).double(), torch.randn(n, r, N, generator=g).double(), torch.randn(b, K, generator=g).double()
    ids = torch.tensor([0, 2, 1, 1, 0])
    whole = torch.einsum("bk,bkr,brn->bn", x, A[ids], B[ids])
    a, c = shard_adapters(A, B, "col", rank, world)
    w = N // world
    assert torch.allclose(torch.einsum("bk,bkr,brn->bn", x, a[ids], c[ids]), whole[:, rank * w:(rank + 1) * w])
    a, c = shard_adapters(A, B, "row", rank, world)
    k = K // world
    part = torch.einsum("bk,bkr,brn->bn", x[:, rank * k:(rank + 1) * k], a[ids], c[ids])
    dist.all_reduce(part)
    assert torch.allclose(part, whole)
    logits = torch.randn(b, 16 * world, generator=g).half()
    got = gather_logits(shard_vocab(logits, rank, world).contiguous(), world)
    assert torch.equal(got, logits)
    with pytest.raises(ValueError, match="split"):
        shard_adapters(A, B, "both", rank, 2)
    dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 4])
def test_sharded_requests(world, monkeypatch):
    monkeypatch.setenv("GLOO_SOCKET_IFNAME", "lo")
    monkeypatch.setenv("OMP_NUM_THREADS", "2")
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_worker, args=(world, port), nprocs=world, join=True)
