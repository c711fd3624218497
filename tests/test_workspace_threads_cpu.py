"""Two threads on one stream: the launches of one call may come between those of another's, so no two
threads' calls share a workspace."""

import threading

import pytest

from hk import _native as nat


@pytest.fixture
def eager(monkeypatch):
    monkeypatch.setattr(nat, "stream_of", lambda device: 7)
    monkeypatch.setattr(nat, "capturing", lambda device: False)
    monkeypatch.setattr(nat, "_WS", {})


def _in_a_thread(f):
    got = []
    t = threading.Thread(target=lambda: got.append(f()))
    t.start()
    t.join()
    return got[0]


def test_threads_have_workspaces_of_their_own(eager):
    mine = nat.workspace("cpu", 4096)
    theirs = _in_a_thread(lambda: nat.workspace("cpu", 4096))
    assert theirs is not mine and theirs.data_ptr() != mine.data_ptr()
    # at the same time, each thread's own is one buffer, grown as the main thread's is
    start = threading.Barrier(4)

    def work():
        start.wait()
        small = nat.workspace("cpu", 64)
        start.wait()
        assert nat.workspace("cpu", 32) is small
        start.wait()
        return small, nat.workspace("cpu", 8192), nat.workspace("cpu", 8192)

    out = []
    threads = [threading.Thread(target=lambda: out.append(work())) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len({x.data_ptr() for o in out for x in o[1:]} | {mine.data_ptr()}) == 5
    assert all(o[1] is o[2] and o[1].numel() * 4 >= 8192 for o in out)
    assert nat.workspace("cpu", 4096) is mine


def test_a_threads_workspaces_end_with_it(eager):
    import gc
    import weakref

    ref = _in_a_thread(lambda: weakref.ref(nat.workspace("cpu", 4096)))
    gc.collect()
    assert ref() is None
