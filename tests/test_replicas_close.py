"""What ReplicaGroup.close waits for on the rank that hosts the store (CPU)."""

import os
import socket
import subprocess
import sys
import time

import pytest

from breeze_b200 import replicas


def host(world=2, failed=()):
    for _ in range(3):  # a port taken by someone else: choose another
        with socket.socket() as s:
            s.bind(("127.0.0.1", 0))
            port = s.getsockname()[1]
        try:
            grp = replicas.ReplicaGroup(0, world, "127.0.0.1", port, timeout_s=3.0, prefix=f"c{port}")
        except RuntimeError:
            continue
        grp.failed |= set(failed)
        return grp
    raise AssertionError("no free port")


@pytest.fixture(autouse=True)
def _own_store(monkeypatch):
    monkeypatch.delenv("TORCHELASTIC_USE_AGENT_STORE", raising=False)


def leave(grp, rank, pid, machine=None):
    """What rank `rank` of process `pid` does when it closes."""
    grp.store.set(grp._key("close", f"left{rank}"), f"{pid} {machine or replicas._machine()}")


def took(grp, **kw):
    t = time.monotonic()
    grp.close(**kw)
    return time.monotonic() - t


def process(seconds):
    return subprocess.Popen([sys.executable, "-S", "-c", f"import time; time.sleep({seconds})"])


def test_nobody_left_to_wait_for():
    assert took(host(failed=[1])) < 0.4
    assert took(host(world=1)) < 0.4


def test_a_process_that_has_ended_is_not_waited_for():
    p = process(0)
    p.wait()
    grp = host()
    leave(grp, 1, p.pid)
    assert took(grp, linger_s=20.0) < 5.0


def test_a_process_that_ends_is_outlived():
    p = process(1.0)
    grp = host(world=3, failed=[2])
    leave(grp, 1, p.pid)
    assert took(grp, linger_s=20.0) < 15.0  # its end, not the limit
    assert os.waitid(os.P_PID, p.pid, os.WEXITED | os.WNOHANG) is not None  # (ended, and not yet waited for)


@pytest.mark.parametrize("limit", [dict(linger_s=0.3), dict(timeout_s=0.3, linger_s=20.0)])
def test_a_process_that_lives_on_costs_the_limit(limit):
    p = process(60)
    try:
        grp = host()
        leave(grp, 1, p.pid)
        assert 0.2 < took(grp, **limit) < 10.0
        assert p.poll() is None
    finally:
        p.kill()
        p.wait()


def test_a_process_of_another_machine_is_not_waited_for():
    grp = host()
    leave(grp, 1, os.getpid(), "elsewhere/1")
    assert took(grp, linger_s=20.0) < 5.0


def test_a_rank_that_does_not_leave_costs_the_timeout_alone():
    assert 0.2 < took(host(), timeout_s=0.3, linger_s=20.0) < 10.0
