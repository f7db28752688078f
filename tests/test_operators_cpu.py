"""Refusals of the decay attention, embedding and sampling entry points, and
their workspace queries (no launches: runs without a GPU)."""

import ctypes

import pytest
import torch

DIMS, UNSUPPORTED, NULL, ALIGN, WORKSPACE = 1, 2, 3, 4, 6
P, ODD = 1 << 20, (1 << 20) + 8  # addresses that no call here reads


def _lib():
    from mamba4_b200 import _lib

    return _lib.load(), _lib.DecayDims


def _decay(batch=2, time=100, heads=4, kv_heads=2, dk=64, dv=128, bf16=1):
    row = (ctypes.c_int64 * 3)
    _, dims = _lib()
    return dims(batch, time, heads, kv_heads, dk, dv, bf16, 0.125, row(time * heads * dk, heads * dk, dk),
                row(time * kv_heads * dk, kv_heads * dk, dk), row(time * kv_heads * dv, kv_heads * dv, dv))


BAD_DIMS = [(dict(batch=0), DIMS), (dict(time=0), DIMS), (dict(heads=0), DIMS), (dict(kv_heads=0), DIMS),
            (dict(kv_heads=3), DIMS), (dict(dk=0), DIMS), (dict(dv=-8), DIMS), (dict(dk=136), UNSUPPORTED),
            (dict(dv=256), UNSUPPORTED), (dict(dk=60), UNSUPPORTED), (dict(batch=65536), UNSUPPORTED)]


@pytest.mark.parametrize("change,status", BAD_DIMS)
def test_decay_dims(change, status):
    lib, _ = _lib()
    d = _decay(**change)
    assert lib.m4_decay_fwd(d, *[P] * 8, P, 1 << 40, None) == status
    assert lib.m4_decay_bwd(d, *[P] * 12, P, 1 << 40, None) == status
    assert lib.m4_decay_fwd_workspace_bytes(d) == lib.m4_decay_bwd_workspace_bytes(d) == 0


def test_decay_pointers_and_workspace():
    lib, _ = _lib()
    d = _decay()
    optional = {"fwd": (4, 5), "bwd": (4, 5, 7, 11)}  # lengths, initial; and d_final, d_initial
    for at in range(8):
        args = [P] * 8
        args[at] = None
        if at not in optional["fwd"]:
            assert lib.m4_decay_fwd(d, *args, P, 1 << 40, None) == NULL, at
    for at in range(12):
        args = [P] * 12
        args[at] = None
        if at not in optional["bwd"]:
            assert lib.m4_decay_bwd(d, *args, P, 1 << 40, None) == NULL, at
    assert lib.m4_decay_fwd(d, *[P] * 8, None, 1 << 40, None) == NULL
    assert lib.m4_decay_fwd(None, *[P] * 8, P, 1 << 40, None) == NULL
    for query, call, n in ((lib.m4_decay_fwd_workspace_bytes, lib.m4_decay_fwd, 8),
                           (lib.m4_decay_bwd_workspace_bytes, lib.m4_decay_bwd, 12)):
        need = query(d)
        assert need > 0
        assert call(d, *[P] * n, P, need - 1, None) == WORKSPACE
    out = [P] * 8
    out[6] = ODD
    assert lib.m4_decay_fwd(d, *out, P, 1 << 40, None) == ALIGN


def test_decay_workspace_grows_with_what_is_kept():
    """Shared heads keep a float32 gradient per query head; few heads and rows
    over a long axis keep their segments' states."""
    lib, _ = _lib()
    own, shared = _decay(kv_heads=4), _decay(kv_heads=2)
    part = 2 * 100 * 4 * (64 + 128) * 4
    assert lib.m4_decay_bwd_workspace_bytes(shared) - lib.m4_decay_bwd_workspace_bytes(own) >= part
    short, long = _decay(batch=1, time=64), _decay(batch=1, time=32768)
    assert lib.m4_decay_fwd_workspace_bytes(long) >= lib.m4_decay_fwd_workspace_bytes(short) + 2 * 4 * 64 * 128 * 4


def test_decay_step():
    lib, _ = _lib()
    for change, status in BAD_DIMS:
        if status == DIMS and "time" not in change or change in (dict(dk=136), dict(dv=256)):
            assert lib.m4_decay_step(_decay(**change), *[P] * 7, None) == status, change
    assert lib.m4_decay_step(_decay(batch=1 << 30), *[P] * 7, None) == UNSUPPORTED
    for at in range(7):
        args = [P] * 7
        args[at] = None
        assert lib.m4_decay_step(_decay(), *args, None) == NULL, at
    assert lib.m4_decay_step(None, *[P] * 7, None) == NULL


def test_embedding():
    lib, _ = _lib()
    for rows, vocab, dim in ((0, 10, 8), (4, 0, 8), (4, 10, 0), (-1, 10, 8)):
        assert lib.m4_embedding_fwd(rows, vocab, dim, P, P, 1, 1.0, P, 1, None) == DIMS
        assert lib.m4_embedding_bwd(rows, vocab, dim, P, P, 1, 1.0, P, 1, P, 1 << 40, None) == DIMS
        assert lib.m4_embedding_workspace_bytes(rows, vocab, dim) == 0
    for at in range(3):
        a = [P] * 3
        a[at] = None
        assert lib.m4_embedding_fwd(4, 10, 8, a[0], a[1], 1, 1.0, a[2], 1, None) == NULL
        assert lib.m4_embedding_bwd(4, 10, 8, a[0], a[1], 1, 1.0, a[2], 1, P, 1 << 40, None) == NULL
    need = lib.m4_embedding_workspace_bytes(4, 10, 8)
    assert need > 0
    assert lib.m4_embedding_bwd(4, 10, 8, P, P, 1, 1.0, P, 1, None, need, None) == NULL
    assert lib.m4_embedding_bwd(4, 10, 8, P, P, 1, 1.0, P, 1, ODD, need, None) == ALIGN
    assert lib.m4_embedding_bwd(4, 10, 8, P, P, 1, 1.0, P, 1, P, need - 1, None) == WORKSPACE
    # (ranges of at most 2048 ids, 1024 of them; 2^28 tokens)
    assert lib.m4_embedding_workspace_bytes(4, 1 << 21, 8) > 0
    for rows, vocab in ((4, (1 << 21) + 1), ((1 << 28) + 1, 10)):
        assert lib.m4_embedding_workspace_bytes(rows, vocab, 8) == 0
        assert lib.m4_embedding_bwd(rows, vocab, 8, P, P, 1, 1.0, P, 1, P, 1 << 40, None) == UNSUPPORTED


def test_sample():
    lib, _ = _lib()

    def call(rows=2, vocab=100, ld=100, logits=P, uniform=P, tokens=P, log_prob=P):
        return lib.m4_sample(rows, vocab, ld, logits, 1, uniform, None, None, None, None, 1.0, 0, 1.0, 0.0, tokens,
                             log_prob, None)

    assert call(rows=0) == call(vocab=0) == call(ld=99) == DIMS
    assert call(vocab=262145, ld=262145) == call(rows=1 << 27) == UNSUPPORTED
    for name in ("logits", "uniform", "tokens", "log_prob"):
        assert call(**{name: None}) == NULL, name


def test_python_entry_points_refuse_cpu_tensors():
    import mamba4_b200 as m4

    q, decay = torch.zeros(1, 2, 2, 8), torch.zeros(2)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        m4.decay_attention(q, q, q, decay)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        m4.decay_attention_step(torch.zeros(1, 2, 8, 8), q[:, 0], q[:, 0], q[:, 0], decay)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        m4.embedding_lookup(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        m4.sample_tokens(torch.zeros(2, 5), torch.zeros(2))


def test_launches_go_to_the_device_of_their_tensors(monkeypatch):
    """The device is current at the call, its own stream is the last argument,
    and the one that was current before is so again (a stand-in for torch's
    device state: runs without a GPU)."""
    import contextlib
    import types

    from mamba4_b200 import _lib

    state = dict(current=0)
    calls = []

    @contextlib.contextmanager
    def device(index):
        before, state["current"] = state["current"], index
        try:
            yield
        finally:
            state["current"] = before

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: state["current"], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    status = dict(value=0)

    def call(*args):
        calls.append((state["current"], args))
        return status["value"]

    monkeypatch.setattr(_lib, "load", lambda: types.SimpleNamespace(m4_sample=call, m4_status_string=lambda s: b"bad"))
    on = lambda index: types.SimpleNamespace(get_device=lambda: index)  # noqa: E731
    _lib.launch(on(0), "m4_sample", 1, 2)
    _lib.launch(on(3), "m4_sample", 5)
    assert calls == [(0, (1, 2, 100)), (3, (5, 103))] and state["current"] == 0
    status["value"] = 2
    with pytest.raises(RuntimeError, match="m4_sample"):
        _lib.launch(on(1), "m4_sample")
    assert state["current"] == 0
