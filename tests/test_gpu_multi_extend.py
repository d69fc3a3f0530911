"""Multi-GPU: ``DWALM.extend`` and ``DWALM.verify`` over a row-sharded pool against the same model
on one GPU.

Runs only when 2 or more CUDA devices are visible.  Every rank calls with the same tokens
in the same order, so the plans' exchanges are made together; the process group has a
short timeout, so a rank that fails ends the others' next collective with an error.
"""
import os

import pytest
import torch

from test_gpu_multi import _free_port

pytestmark = pytest.mark.gpu


def _worker(rank, world, port, q):
    from datetime import timedelta

    import torch.distributed as dist

    import computd_b200 as cb
    from computd_b200.dwa_lm import DWALM, DWALMConfig

    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    os.environ.setdefault("NCCL_NVLS_ENABLE", "0")
    torch.cuda.set_device(rank)
    dev = torch.device("cuda", rank)
    dist.init_process_group("nccl", rank=rank, world_size=world, timeout=timedelta(seconds=60), device_id=dev)
    try:
        msg = "ok"
        g0 = dist.new_group([0])  # every rank takes part in group creation
        for r in (0, 2):
            cfg = DWALMConfig(vocab=65, d_model=64, n_layers=2, n_heads=4, seq_len=64, batch=2,
                              pool_rows=8192, top_k=8, S=2, d_k=32, r=r)

            def pools(rows, off):
                if r:
                    return None, cb.new_normal(rows, cfg.D, seed=71, stddev=0.3, row_offset=off, device=dev)
                return (cb.new_normal(rows, cfg.key_width, seed=72, stddev=cfg.key_width ** -0.5, row_offset=off,
                                      device=dev),
                        cb.new_normal(rows, cfg.d_model, seed=73, stddev=cfg.d_model ** -0.5, row_offset=off,
                                      device=dev))

            spec = cb.ShardSpec(cfg.pool_rows, rank, world)
            lm = DWALM(cfg, *pools(spec.n_local, spec.row_begin))
            one = DWALM(cfg, *pools(cfg.pool_rows, 0), group=g0) if rank == 0 else None
            i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
            tokens = torch.randint(0, cfg.vocab, (2, 40), device=dev,
                                   generator=torch.Generator(device=dev).manual_seed(3))
            caches = [m.new_cache(8, page_size=16) if m is not None else None for m in (lm, one)]
            table = i32([[3, 0, 5, 7], [1, 6, 2, 4]])
            at = 0
            for n in (20, 1, 1, 7):  # row counts 40, 2, 2, 14
                at += n
                a = (tokens[:, at - n:at].reshape(-1), table, i32([at] * 2))
                got = lm.extend(a[0], caches[0], *a[1:])
                if rank == 0:
                    want = one.extend(a[0], caches[1], *a[1:])
                    torch.cuda.synchronize()
                    err, size = float((got.float() - want.float()).abs().max()), float(want.float().abs().max())
                    if msg == "ok" and not err <= 2e-2 * size:
                        msg = f"r={r}, {n} tokens: sharded extend differs by {err:.3g} of {size:.3g}"
            drafts = i32([[1, 2, 3], [4, 5, 6]])
            u, s = torch.zeros((2, 3), device=dev), torch.full((2,), 0.5, device=dev)
            accepted, _, new = lm.verify(i32([7, 8]), drafts, None, u, s, caches[0], table, i32([at] * 2))
            torch.cuda.synchronize()
            if msg == "ok" and (accepted.tolist() != [3, 3] or new.tolist() != [at + 4] * 2):
                msg = f"r={r}: sharded verify accepted {accepted.tolist()}"
            caches[0].check()
            status = lm.status()
            if msg == "ok" and status != 0:
                msg = f"r={r}: status {status}"
            lm.close()
        q.put((rank, msg))
        dist.barrier(device_ids=[rank])
    finally:
        dist.destroy_process_group()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs 2 GPUs")
@pytest.mark.parametrize("world", [2, 4])
def test_sharded_extend_matches_single_gpu(world):
    if torch.cuda.device_count() < world:
        pytest.skip(f"needs {world} GPUs")
    import torch.multiprocessing as mp

    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    results = [q.get(timeout=300) for _ in range(world)]
    for p in procs:
        p.join(timeout=120)
        assert p.exitcode == 0
    for rank, msg in sorted(results):
        assert msg == "ok", f"rank {rank}: {msg}"
