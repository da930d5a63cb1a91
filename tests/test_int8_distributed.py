"""precision="int8" with max_grad_norm on two ranks (gloo): equal directions,
equal bounds, equal parameters."""
import os
import tempfile

import torch
import torch.multiprocessing as mp

from distributedes_amd import preset


def _train(rank, world, store, q):
    if world > 1:
        os.environ.update(DES_FILE_STORE=store, WORLD_SIZE=str(world),
                          RANK=str(rank), LOCAL_RANK=str(rank))
    try:
        from distributedes_amd.core.engine import TrainState, train_step
        st = TrainState(preset(
            "cartpole_es", pop=8, generations=3, episode_steps=15,
            noise_table_size=1 << 16, device="cpu", backend="gloo",
            precision="int8", max_grad_norm=0.5, log_every=10 ** 9),
            ops_backend="torch_ref")
        norms = [train_step(st)["grad_norm"] for _ in range(3)]
        q.put((rank, "ok", st.theta.tolist(), norms))
    except Exception:  # pragma: no cover
        import traceback
        q.put((rank, traceback.format_exc(), None, None))
    finally:
        import torch.distributed as dist
        if dist.is_initialized():
            dist.destroy_process_group()


def test_two_ranks_take_the_same_steps():
    store = os.path.join(tempfile.mkdtemp(prefix="des_store_"), "store")
    ctx = mp.get_context("spawn")
    q = ctx.SimpleQueue()
    procs = [ctx.Process(target=_train, args=(r, 2, store, q))
             for r in range(2)]
    for p in procs:
        p.start()
    got = {}
    for _ in procs:
        rank, status, theta, norms = q.get()
        assert status == "ok", status
        got[rank] = (theta, norms)
    for p in procs:
        p.join(timeout=60)
    assert got[0] == got[1]
    # one rank alone: the same members, the sum of their estimates in other order
    one = ctx.SimpleQueue()
    p = ctx.Process(target=_train, args=(0, 1, store, one))
    p.start()
    _, status, theta, norms = one.get()
    assert status == "ok", status
    p.join(timeout=60)
    torch.testing.assert_close(torch.tensor(theta), torch.tensor(got[0][0]),
                               rtol=1e-4, atol=1e-5)
