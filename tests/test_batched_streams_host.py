"""The order of streams and events in DecodeBatch, on stand-ins for the library, the streams
and the events (no GPU needed): plain and drafted layers go through one and the same
resolve-and-gather step, whose waits protect the hot rows and the shared miss lists."""

from types import SimpleNamespace

import pytest
import torch

from hisparse_b200 import _lib, batched, tree


class Place:
    shape = (8, 2)

    def data_ptr(self):
        return 16


@pytest.fixture
def world(monkeypatch):
    log = []

    class Stream:
        def __init__(self, name):
            self.name, self.cuda_stream = name, name

        def wait_event(self, event):
            log.append((self.name, "wait", event.name))

    class Event:
        made = 0

        def __init__(self, *args, **kwargs):
            Event.made += 1
            self.name = f"event{Event.made}"

        def record(self, stream):
            log.append((stream.name, "record", self.name))

    class Library:
        def __getattr__(self, name):
            def call(*args):
                stream = next(a for a in reversed(args) if a in ("compute", "transfer"))
                log.append((stream, name))
                return 0
            return call

    batch = object.__new__(batched.DecodeBatch)
    place = Place()
    for name in ("physical", "miss_host", "miss_device", "ready", "status", "tokens"):
        setattr(batch, name, place)
    batch.resolve_ws = batch.attend_ws = None
    batch.resolve_ws_bytes = batch.attend_ws_bytes = batch._dtype = batch._row_bytes = 0
    batch.batch, batch.width, batch.q_heads, batch.hot_rows = 2, 64, 4, 64
    batch.device, batch.group = torch.device("cpu"), None
    batch.compute, batch.transfer = Stream("compute"), Stream("transfer")
    batch.config = SimpleNamespace(head_dim=8, kv_heads=2, page_size=16)
    batch.cache = SimpleNamespace(hot_blocks=4, mapped=place, host=place, pool=place)
    last, ready = Event(), Event()
    last.name, ready.name = "last readers", "last gather"
    names = ("src_ptrs", "res_ptrs", "hot_ptrs", "tag_ptrs", "lru_ptrs", "lengths", "counts")
    batch.layers = [SimpleNamespace(**{n: place for n in names}, table_pages=4, ready=ready,
                                    last_use=last)]
    monkeypatch.setattr(_lib, "load", Library)
    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: batch.compute)
    monkeypatch.setattr(tree, "attend_tree",
                        lambda *a, **k: log.append(("compute", "attend_tree")))
    return batch, log


def run(batch, log, drafted):
    positions = torch.zeros((2, 64), dtype=torch.int32)
    if drafted:
        batch.layer_tree(0, torch.zeros(2, 3, 4, 8), None, None, None, None, positions, None)
    else:
        batch.layer(0, torch.zeros(2, 4, 8), positions=positions)
    return log


@pytest.mark.parametrize("drafted", [False, True])
def test_gather_waits_for_the_resolver_and_the_last_readers(world, drafted):
    batch, log = world
    run(batch, log, drafted)
    resolve = log.index(("compute", "hs_resolve_rows_batched"))
    gather = log.index(("transfer", "hs_gather_rows"))
    assert ("compute", "wait", "last gather") in log[:resolve]
    _, _, resolved = log[resolve + 1]
    assert log[resolve + 1] == ("compute", "record", resolved)
    assert log[resolve + 2:gather] == [("transfer", "wait", resolved),
                                       ("transfer", "wait", "last readers")]
    assert log[gather + 1][:2] == ("transfer", "record")
    ready = log[gather + 1][2]
    waits = log.index(("compute", "wait", ready))
    readers = [i for i, entry in enumerate(log) if "attend" in entry[1]]
    assert readers[-1] > waits and (not drafted or readers[0] > waits)
    assert log[-1][:2] == ("compute", "record")  # the new last readers


@pytest.mark.parametrize("drafted", [False, True])
def test_one_resolve_and_gather_step(world, drafted, monkeypatch):
    batch, log = world
    step, calls = batched.DecodeBatch._resolve_and_gather, []

    def spy(self, *args, **kwargs):
        calls.append(len(log))
        return step(self, *args, **kwargs)

    monkeypatch.setattr(batched.DecodeBatch, "_resolve_and_gather", spy)
    run(batch, log, drafted)
    assert len(calls) == 1 and log[calls[0]] == ("compute", "hs_resolve_rows_batched")
    assert [e[1] for e in log].count("hs_gather_rows") == 1
