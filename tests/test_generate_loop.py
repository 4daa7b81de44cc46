"""PFlashDecoder.generate's loop on the CPU; the model and the draw are stand-ins.
Over column-parallel ranks (two gloo ones) every rank takes the first rank's
tokens, whatever its own generator's state is; a cache that is too small loses
nothing that was drawn."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

V = 50


def _free_port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def _logits(ids):
    return torch.randn(len(ids), V, generator=torch.Generator().manual_seed(int(ids.sum())))


def _draw(logits, u, temperature, top_k, top_p, min_p):
    """A token of the whole range, by the uniform number alone."""
    return (u * V).long()


def _decoder(decode, tp, fed):
    d = object.__new__(decode.PFlashDecoder)
    d.tp, d._graph, d.device, d.max_seq, d.length = tp, None, torch.device("cpu"), 64, 0

    def forward(ids):
        fed.append(ids.tolist())
        if tp is not None:
            tp.gather([torch.zeros(1, 3)])  # a projection's: a rank that left the loop would be missed here
        if d.length + len(ids) > d.max_seq:
            raise ValueError("cache")
        d.length += len(ids)
        return _logits(ids)

    d.forward = forward
    return d


def _worker(rank, world, port, eos, out_q):
    import sys
    from datetime import timedelta

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path[:0] = [root, os.path.join(root, "polar-flash_b200")]
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=timedelta(seconds=30))
    try:
        from polarflash_b200 import decode
        from polarflash_b200.parallel import GroupGather

        decode.sample_logits = _draw
        fed = []
        d = _decoder(decode, GroupGather(), fed)
        gen = torch.Generator().manual_seed(7 + rank)  # a seed per rank
        alone = (torch.rand(12, generator=torch.Generator().manual_seed(7 + rank)) * V).long().tolist()
        out_q.put((rank, d.generate(torch.tensor([3, 1, 4]), 12, eos=eos, generator=gen), fed, alone))
        dist.barrier()
    finally:
        dist.destroy_process_group()


def _run(eos):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, eos, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = sorted(q.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    return res


def test_ranks_with_different_generators_draw_the_same_tokens():
    (_, a, fed_a, alone), (_, b, fed_b, other) = _run(None)
    assert a == b == alone and a != other
    assert fed_a == fed_b == [[3, 1, 4]] + [[t] for t in a[:-1]]
    eos = a[4]
    (_, a2, fed_a, _), (_, b2, fed_b, _) = _run(eos)  # both leave the loop at once
    assert a2 == b2 == a[: a.index(eos) + 1] and fed_a == fed_b


def test_where_the_cache_ends(monkeypatch):
    from polarflash_b200 import decode

    monkeypatch.setattr(decode, "sample_logits", _draw)
    gen = lambda: torch.Generator().manual_seed(3)  # noqa: E731
    fed = []
    want = _decoder(decode, None, []).generate(torch.arange(10), 55, generator=gen())
    assert len(want) == 55  # 10 + 54 cached
    d = _decoder(decode, None, fed)
    with pytest.raises(ValueError):
        d.generate(torch.arange(10), 56, generator=gen())
    assert fed == [] and d.length == 0
    never = next(t for t in range(V + 1) if t not in want)
    assert d.generate(torch.arange(10), 100, eos=never, generator=gen()) == want and d.length == 64
