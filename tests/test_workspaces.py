"""Workspaces of attention calls: kept per thread, device and stream."""

import threading

import pytest
import torch as t

from aiproj_amd.kernals import decode_attention


@pytest.fixture
def workspace(monkeypatch):
    monkeypatch.setattr(t.cuda, "is_current_stream_capturing", lambda: False)
    return lambda stream, nbytes: decode_attention._workspace(t.device("cpu"), stream, nbytes)


def _in_thread(fn):
    got = []
    thread = threading.Thread(target=lambda: got.append(fn()))
    thread.start()
    thread.join()
    return got[0]


def test_one_thread_reuses_its_block(workspace):
    first = workspace(7, 100)
    assert workspace(7, 60) is first and workspace(8, 60) is not first
    assert workspace(7, 200).numel() == 200 and workspace(7, 100).numel() == 200


def test_threads_have_blocks_of_their_own(workspace):
    """A call's launches are enqueued without the interpreter's lock: another thread's may come in between."""
    mine = workspace(7, 100)
    theirs = _in_thread(lambda: workspace(7, 100))
    assert mine.data_ptr() != theirs.data_ptr()
    assert workspace(7, 100) is mine
