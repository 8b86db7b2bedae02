"""Dropout's numbers and the refusals of the norm and dropout entry points, without a GPU."""
import ctypes
import threading

import numpy as np
import pytest
import torch

import _draw
from easyllm_amd import _lib, dropout
from easyllm_amd.checkpointing import checkpoint


def test_the_restated_generator_gives_the_published_vectors():
    """Known answers of Philox-4x32-10 that its authors publish with the method."""
    for counter, key, want in [
            ([0] * 4, [0] * 2, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
            ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
            ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0], [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1])]:
        got = _draw.philox([np.array([c], dtype=np.uint64) for c in counter], key)
        assert [int(w[0]) for w in got] == want


def test_the_shares_dropped_and_the_expected_value():
    n = _draw.numbers(0, 1 << 17, 99, 3).ravel()
    for t in (655, 6554, 32768):
        share = (n < t).mean()
        assert abs(share - t / 65536) < 5 * (t / 65536 / n.size) ** 0.5
    assert (_draw.numbers(5, 8, 99, 3) == _draw.numbers(0, 16, 99, 3)[5:13]).all()


def test_thresholds():
    assert [dropout.threshold_of(p) for p in (0.0, 0.1, 0.5, 1.0, 1e-6, 1 - 1e-6)] == [0, 6554, 32768, 65536, 0, 65536]
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            dropout.threshold_of(p)


def test_draws_count_up_and_can_be_restored():
    kept = dropout.get_state()
    try:
        dropout.manual_seed(7)
        first = [dropout.next_draw() for _ in range(3)]
        assert first == [(7, 0, None), (7, 1, None), (7, 2, None)]
        state = dropout.get_state()
        more = [dropout.next_draw() for _ in range(2)]
        dropout.set_state(state)
        assert [dropout.next_draw() for _ in range(2)] == more
        dropout.set_state((7, 2 ** 32))
        assert dropout.next_draw()[:2] == (8, 0)  # (offsets have 32 bits)
    finally:
        dropout.set_state(kept)


def test_recorded_draws_are_replayed_nested_and_by_thread():
    with dropout.recording() as outer:
        a = dropout.next_draw()
        with dropout.recording() as inner:
            b = dropout.next_draw()
        c = dropout.next_draw()
    assert outer == [a, b, c] and inner == [b]
    elsewhere = []
    with dropout.replaying(outer), dropout.recording() as again:
        t = threading.Thread(target=lambda: elsewhere.append(dropout.next_draw()))
        t.start()
        t.join()
        assert [dropout.next_draw() for _ in range(3)] == outer
        with pytest.raises(RuntimeError):
            dropout.next_draw()
    assert again == outer and elsewhere[0] not in outer


def test_a_checkpointed_chunk_draws_again_what_it_drew(monkeypatch):
    """Through the framework's checkpoint: the recomputed forward sees the forward's numbers, whatever was drawn in between, also in chunks inside chunks."""
    seen = []

    def layer(x):
        seen.append(dropout.next_draw())
        return x * seen[-1].offset

    x = torch.ones(3, requires_grad=True)
    y = checkpoint(lambda v: layer(checkpoint(layer, layer(v))), x)
    drawn = list(seen)
    dropout.next_draw()
    y.sum().backward()
    assert len(drawn) == 3 and seen[3:6] == drawn
    assert seen[6:] == [drawn[1]]  # (the inner chunk once more, in its own backward)
    assert torch.equal(x.grad, torch.full((3,), float(drawn[0].offset * drawn[1].offset * drawn[2].offset)))


# ---- refusals: nothing is launched -----------------------------------------------------------------------------------
A = 1 << 20  # an aligned address nobody reads


def refused(code, text, name, *args):
    _lib.load()
    with pytest.raises(RuntimeError, match=r"\(%d\).*%s" % (code, text)):
        _lib.call(name, *args)


def drop(share=6554, step=None):
    return ctypes.byref(_lib.Dropout(1, 2, share, step))


def grad(f32=None, bf16=None):
    return ctypes.byref(_lib.LayerGrad(f32, bf16, 0))


def test_dropout_add_refuses():
    fwd = lambda x=A, b=None, r=None, d=None, o=A, rows=2, n=64: ("ezl_dropout_add_fwd", x, b, r, d, o, rows, n, None)  # noqa: E731
    for args in (dict(n=60), dict(n=0), dict(rows=-1), dict(rows=2 ** 31 - 1), dict(n=2 ** 31)):
        refused(-2, "n % 8", *fwd(**args))
    for args in (dict(x=None), dict(o=None)):
        refused(-1, "null", *fwd(**args))
    for args in (dict(x=A + 2), dict(b=A + 8), dict(r=A + 4), dict(o=A + 2)):
        refused(-1, "aligned", *fwd(**args))
    refused(-1, "drop_of_65536", *fwd(d=drop(65537)))
    refused(-1, "drop_of_65536", *fwd(d=drop(-1)))
    refused(-1, "step", *fwd(d=drop(step=A + 4)))
    bwd = lambda dy=A, d=None, dx=A, g=None, ws=None, size=0: ("ezl_dropout_add_bwd", dy, d, dx, g, ws, size, 2, 64, None)  # noqa: E731
    refused(-1, "null", *bwd(dy=None, d=drop()))
    refused(-1, "null", *bwd(dx=None, d=drop()))
    refused(-1, "without drop", *bwd(g=grad(f32=A), ws=A, size=1 << 20))
    refused(-1, "nothing to do", *bwd(dx=None))
    refused(-1, "workspace", *bwd(d=drop(), g=grad(f32=A)))
    refused(-1, "workspace", *bwd(dx=None, g=grad(bf16=A), ws=A, size=_lib.column_sum_workspace_bytes(2, 64) - 1))
    refused(-1, "aligned", *bwd(dx=None, g=grad(bf16=A), ws=A + 4, size=1 << 20))


def test_column_sums_of_more_columns_than_a_launch_has_threads_for_are_refused():
    n = 2 ** 27 + 8
    refused(-2, "column sums", "ezl_dropout_add_bwd", A, drop(), A, grad(f32=A), A, 1 << 50, 1, n, None)
    refused(-2, "column sums", "ezl_act_bwd", 1, A, A, A, grad(bf16=A), A, 1 << 50, 1, n, None)


def test_norm_refuses():
    def fwd(kind=0, x=A, xb=None, r=None, d=None, w=A, b=None, y=A, s=None, mean=A, rstd=A, rows=2, h=64):
        return ("ezl_norm_fwd", kind, x, xb, r, d, w, b, y, s, mean, rstd, rows, h, 1e-5, None)
    refused(-1, "kind", *fwd(kind=2))
    for args in (dict(h=60), dict(h=0), dict(h=8200), dict(rows=-1), dict(rows=2 ** 31 - 1)):
        refused(-2, "h % 8", *fwd(**args))
    for args in (dict(x=None), dict(w=None), dict(y=None), dict(rstd=None), dict(mean=None)):
        refused(-1, "null", *fwd(**args))
    refused(-1, "sum_out", *fwd(r=A))
    refused(-1, "sum_out", *fwd(s=A))
    for args in (dict(xb=A), dict(d=drop()), dict(kind=1)):
        refused(-1, "residual", *fwd(**args))
    refused(-1, "no bias", *fwd(kind=1, r=A, s=A, b=A))
    refused(-1, "drop_of_65536", *fwd(r=A, s=A, d=drop(70000)))
    for args in (dict(x=A + 2), dict(w=A + 8), dict(y=A + 4), dict(b=A + 2), dict(r=A + 2, s=A), dict(r=A, s=A + 2), dict(r=A, s=A, xb=A + 2)):
        refused(-1, "aligned", *fwd(**args))

    size = _lib.norm_bwd_workspace_bytes(2, 64)

    def bwd(kind=0, dy=A, ds=None, s=A, w=A, mean=A, rstd=A, d=None, dx=A, dr=None, gw=grad(f32=A), gb=None, gx=None, ws=A, size=size, rows=2, h=64):
        return ("ezl_norm_bwd", kind, dy, ds, s, w, mean, rstd, d, dx, dr, gw, gb, gx, ws, size, rows, h, None)
    refused(-1, "kind", *bwd(kind=-1))
    for args in (dict(h=60), dict(h=8200), dict(rows=2 ** 31 - 1)):
        refused(-2, "h % 8", *bwd(**args))
    for args in (dict(dy=None), dict(s=None), dict(w=None), dict(mean=None), dict(rstd=None), dict(dx=None)):
        refused(-1, "null", *bwd(**args))
    for args in (dict(gw=None), dict(gw=grad())):
        refused(-1, "dweight", *bwd(**args))
    refused(-1, "no bias", *bwd(kind=1, gb=grad(bf16=A)))
    refused(-1, "go together", *bwd(d=drop()))
    refused(-1, "go together", *bwd(dr=A))
    refused(-1, "workspace", *bwd(ws=None))
    refused(-1, "workspace", *bwd(size=size - 1))
    for args in (dict(dy=A + 2), dict(ds=A + 2), dict(s=A + 8), dict(w=A + 2), dict(dx=A + 2), dict(d=drop(), dr=A + 2), dict(ws=A + 4)):
        refused(-1, "aligned", *bwd(**args))
