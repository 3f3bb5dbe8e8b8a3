"""Rank-failure detection with store heartbeats: in-process over a HashStore, and across gloo ranks on the CPU."""

import json
import os
import subprocess
import sys
import time

import pytest
import torch.distributed as dist

from astrai_b200.parallel.watchdog import Heartbeat, RankFailure

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_missing_beats_and_announced_exit_are_detected():
    store = dist.HashStore()
    seen = []
    a = Heartbeat(0, 3, store=store, timeout_s=0.3, interval_s=0.05, on_failure=seen.extend).start()
    b = Heartbeat(1, 3, store=store, timeout_s=0.3, interval_s=0.05).start()
    c = Heartbeat(2, 3, store=store, timeout_s=0.3, interval_s=0.05).start()
    try:
        for step in range(1, 4):
            for h in (a, b, c):
                h.beat(step)
            time.sleep(0.05)
        a.check()  # everyone alive
        c.leave("done")  # an orderly exit is seen at the next scan, long before the timeout
        time.sleep(0.2)
        with pytest.raises(RankFailure) as exc:
            a.check()
        assert exc.value.ranks == [2] and "announced" in str(exc.value)
        b.stop()  # rank 1 goes silent: seen after the timeout
        deadline = time.time() + 3
        while 1 not in a.scan() and time.time() < deadline:
            a.beat()
            time.sleep(0.05)
        with pytest.raises(RankFailure) as exc:
            a.check()
        assert exc.value.ranks == [1, 2]
        while 1 not in seen and time.time() < deadline:
            time.sleep(0.01)  # the scanning thread records a dead rank first and calls on_failure right after
        assert sorted(seen) == [1, 2]
    finally:
        for h in (a, b, c):
            h.stop()


@pytest.mark.parametrize("mode", ["leave", "silent"])
def test_survivors_stop_between_steps_when_a_rank_goes_away(tmp_path, mode):
    out = str(tmp_path / "hb.json")
    from helpers import launch_ranks

    code, log = launch_ranks(3, os.path.join(ROOT, "tests", "workers", "heartbeat_ranks.py"), ["--out", out, "--victim", "1", "--mode", mode],
                             29790 if mode == "leave" else 29791, timeout=300, cwd=ROOT)
    assert code == 0, log
    res = {r: json.load(open(f"{out}.{r}")) for r in range(3)}
    assert res[1]["left_at"] == 4 and res[1]["steps"] == 3
    for r in (0, 2):
        assert res[r]["detected"] == [1], res  # found on the host, before the next collective was issued
        assert res[r]["steps"] == 3
        assert res[r]["seconds"] < (1.5 if mode == "leave" else 6.0)


@pytest.mark.parametrize("mode", ["fsdp", "ddp"])
def test_survivors_write_an_emergency_checkpoint_without_collectives(tmp_path, mode):
    """Three gloo ranks train through the real Trainer; rank 1 exits silently between steps.  The survivors must
    return within a bound (no barrier, no gather that waits for the dead rank) and leave the weights on disk."""
    out, ckpt = str(tmp_path / "res"), str(tmp_path / "ckpt")
    from helpers import launch_ranks

    code, log = launch_ranks(3, os.path.join(ROOT, "tests", "workers", "rank_loss_trainer.py"), ["--out", out, "--ckpt", ckpt, "--mode", mode],
                             29793 if mode == "fsdp" else 29794, timeout=300, cwd=ROOT)
    assert code == 0, log
    gone = float(open(out + ".gone").read())
    for r in (0, 2):
        res = json.load(open(f"{out}.{r}"))
        assert 1 in res["failure"], res
        assert res["returned_at"] - gone < 20.0, res  # heartbeat timeout 1.5 s + save; far below any process-group timeout
    dirs = [d for d in os.listdir(ckpt) if d.startswith("epoch_") and not d.endswith(".shards")]
    assert len(dirs) == 1
    root = os.path.join(ckpt, dirs[0])
    meta = json.load(open(os.path.join(root, "meta.json")))
    assert meta["emergency"] is True and 1 in meta["failed_ranks"]
    assert os.path.getsize(os.path.join(root, "model.safetensors")) > 0
    if mode == "fsdp":  # sharded optimizer state: one file per survivor, none gathered
        shards = sorted(os.listdir(root + ".shards"))
        assert shards == ["optimizer.rank0.pt", "optimizer.rank2.pt"]
        assert not os.path.exists(os.path.join(root, "optimizer.pt"))
    else:
        assert os.path.getsize(os.path.join(root, "optimizer.pt")) > 0


def test_a_rank_leaves_in_order_when_the_rank_that_hosts_the_store_left_first():
    class Gone:
        def set(self, key, value):
            raise dist.DistNetworkError("Broken pipe")

    Heartbeat(2, 3, store=Gone()).leave("finished")


def test_a_rank_that_leaves_over_a_lost_rank_names_it():
    """Rank 0 finds rank 1 silent and leaves; rank 2, whose own scan sees rank 0's exit first, learns of both."""
    store = dist.HashStore()
    a, b, c = (Heartbeat(r, 3, store=store, timeout_s=t) for r, t in ((0, 0.05), (1, 60.0), (2, 60.0)))
    for h in (a, b, c):
        h.beat(1)
    time.sleep(0.1)
    c.beat(2)
    assert list(a.scan()) == [1]
    a.leave("a rank was lost")
    assert sorted(c.scan()) == [0, 1]
    with pytest.raises(RankFailure) as exc:
        c.check()
    assert exc.value.ranks == [0, 1] and "was lost before rank 0 left" in str(exc.value)


def test_a_report_names_only_ranks_that_went_silent_and_yields_to_what_the_rank_says_itself():
    """A rank that finished is not reported as lost, and a rank that beat after it was given up for lost is believed."""
    store = dist.HashStore()
    a, b, c, d = (Heartbeat(r, 4, store=store, timeout_s=t) for r, t in ((0, 0.05), (1, 60.0), (2, 60.0), (3, 60.0)))
    for h in (a, b, c, d):
        h.beat(1)
    b.leave("finished")
    time.sleep(0.1)
    c.beat(2)
    assert sorted(a.scan()) == [1, 3]  # one has finished, one is silent
    a.leave("a rank was lost")
    time.sleep(0.01)
    d.beat(2)  # it was only slow
    got = c.scan()
    assert sorted(got) == [0, 1] and got[1] == "announced its exit (finished)"
    d.leave("finished")
    assert c.scan()[3] == "announced its exit (finished)"


def test_a_report_is_handed_on():
    """Rank 0 finds rank 1 silent, rank 2 learns of it from rank 0, rank 3 from rank 2 alone."""
    store = dist.HashStore()
    a, b, c, d = (Heartbeat(r, 4, store=store, timeout_s=t) for r, t in ((0, 0.05), (1, 60.0), (2, 60.0), (3, 60.0)))
    for h in (a, b, c, d):
        h.beat(1)
    time.sleep(0.1)
    c.beat(2), d.beat(2)
    assert sorted(a.scan()) == [1]
    a.leave("error")
    assert sorted(c.scan()) == [0, 1]
    store.delete_key("hb/0")
    c.leave("error")
    assert sorted(d.scan()) == [1, 2] and "was lost before rank 2 left" in d.scan()[1]


def test_the_first_exit_that_a_rank_announces_stands():
    store = dist.HashStore()
    a, b = (Heartbeat(r, 2, store=store) for r in range(2))
    a.beat(1), b.beat(1)
    b.leave("error")
    b.leave("finished")
    assert a.scan()[1] == "announced its exit (error)"


@pytest.mark.parametrize("lost", ["silent", "error"])
def test_the_rank_that_hosts_the_store_waits_for_the_survivors(lost):
    import threading

    store = dist.HashStore()
    a, b, c, d = (Heartbeat(r, 4, store=store, timeout_s=2.0) for r in range(4))
    for h in (a, b, c, d):
        h.beat(1)
    if lost == "error":
        b.leave("error")
    else:
        time.sleep(2.1)
        for h in (a, c, d):
            h.beat(2)
    assert sorted(a.scan()) == [1]
    a.leave("a rank was lost")
    threading.Timer(0.15, c.leave, ["a rank was lost"]).start()
    threading.Timer(0.3, d.leave, ["a rank was lost"]).start()
    start = time.time()
    a.outlast_survivors()
    assert 0.25 < time.time() - start < 1.5  # until the last of them has left, not until the timeout
    start = time.time()
    c.outlast_survivors()  # a rank that hosts nothing does not wait
    assert time.time() - start < 1.0


def test_the_wait_for_survivors_ends_with_one_that_is_lost_meanwhile_and_at_the_timeout():
    store = dist.HashStore()
    a, b, c = (Heartbeat(r, 3, store=store, timeout_s=3.0) for r in range(3))
    for h in (a, b, c):
        h.beat(1)
    b.leave("error")
    time.sleep(2.0)
    assert sorted(a.scan()) == [1]
    start = time.time()
    a.outlast_survivors()  # rank 2 has been silent for 2 s: it is lost a second from now
    assert 0.8 < time.time() - start < 2.5 and sorted(a.dead_ranks()) == [1, 2]
    store = dist.HashStore()
    a, b, c = (Heartbeat(r, 3, store=store, timeout_s=t) for r, t in ((0, 0.3), (1, 60.0), (2, 60.0)))
    for h in (a, b, c):
        h.beat(1)
    b.leave("error")
    a.scan()
    c._publish = lambda: store.set("hb/2", f"1 {time.time() + 100:.3f}")  # alive, and never leaving
    c._publish()
    start = time.time()
    a.outlast_survivors()
    assert 0.25 < time.time() - start < 5.0


def test_ranks_that_finish_in_order_are_not_waited_for():
    store = dist.HashStore()
    a, b, c = (Heartbeat(r, 3, store=store, timeout_s=60.0) for r in range(3))
    for h in (a, b, c):
        h.beat(1)
    b.leave("finished")
    assert sorted(a.scan()) == [1]
    a.leave("finished")
    start = time.time()
    a.outlast_survivors()
    assert time.time() - start < 5.0
