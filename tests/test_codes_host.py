"""Learned-code operators (embedding, layer norm, dropout): what they refuse, before anything touches a GPU."""
import ctypes
import itertools

import pytest
import torch

from torch_nerf.amd import _lib, layers, ops

OK, ARG = 0, 1
F32, BF16, F16 = 0, 1, 2
_one = ctypes.c_double(0.0)
P = ctypes.cast(ctypes.pointer(_one), ctypes.c_void_p)      # any non-null address: never dereferenced


def test_layernorm_entries_refuse():
    lib = _lib.load()
    call = lib.nerf_layernorm
    assert call(P, 8, 3, 4, 8, P, P, F32, 1e-5, P, P, P, None) == ARG and b"dtype" in lib.nerf_amd_last_error()
    assert call(P, 8, F16, 4, 8, P, P, BF16, 1e-5, P, P, P, None) == ARG
    assert call(P, 8, F32, 4, 8, P, P, F16, 1e-5, P, P, P, None) == ARG
    assert call(P, 8, F32, -1, 8, P, P, F32, 1e-5, P, P, P, None) == ARG
    assert call(P, 8, F32, 4, 0, P, P, F32, 1e-5, P, P, P, None) == ARG
    assert call(P, 8, F32, 1 << 62, 8, P, P, F32, 1e-5, P, P, P, None) == ARG
    assert call(P, 1 << 25, F32, 4, (1 << 24) + 1, P, P, F32, 1e-5, P, P, P, None) == ARG
    assert call(P, 7, F32, 4, 8, P, P, F32, 1e-5, P, P, P, None) == ARG and b"overlap" in lib.nerf_amd_last_error()
    for eps in (-1e-5, float("nan"), float("inf")):
        assert call(P, 8, F32, 4, 8, P, P, F32, eps, P, P, P, None) == ARG
    assert call(None, 8, F32, 4, 8, P, P, F32, 1e-5, P, P, P, None) == ARG
    assert call(P, 8, F32, 4, 8, P, P, F32, 1e-5, None, P, P, None) == ARG
    assert call(None, 8, F32, 0, 8, None, None, F32, 1e-5, None, None, None, None) == OK       # no rows: nothing to do
    back = lib.nerf_layernorm_backward
    assert back(P, 8, P, 8, 5, 4, 8, P, F32, P, P, P, P, P, P, None) == ARG
    assert back(P, 8, P, 8, F32, 4, 8, P, BF16, P, P, P, P, P, P, None) == ARG
    assert back(P, 7, P, 8, F32, 4, 8, P, F32, P, P, P, P, P, P, None) == ARG
    assert back(P, 8, P, 8, F32, 9000, 8, P, F32, P, P, P, P, P, None, None) == ARG and b"workspace" in lib.nerf_amd_last_error()
    assert back(P, 8, P, 8, F32, 4, 8, P, F32, None, P, P, P, P, P, None) == ARG
    assert lib.nerf_layernorm_backward_workspace_bytes(4, 0, F32) == -1
    assert lib.nerf_layernorm_backward_workspace_bytes(-1, 4, F32) == -1
    assert lib.nerf_layernorm_backward_workspace_bytes(4, 4, 9) == -1
    assert lib.nerf_layernorm_backward_workspace_bytes(4, 64, F16) == 0          # a few rows: one workgroup
    assert lib.nerf_layernorm_backward_workspace_bytes(100000, 64, F32) >= 2 * 64 * 4


def test_embedding_entries_refuse():
    lib = _lib.load()
    call = lib.nerf_embedding
    assert call(P, 10, 8, 3, 8, P, 8, 4, 1.0, P, None) == ARG
    assert call(P, 10, 8, F32, 8, P, 2, 4, 1.0, P, None) == ARG and b"4 or 8" in lib.nerf_amd_last_error()
    assert call(P, 10, 7, F32, 8, P, 8, 4, 1.0, P, None) == ARG
    assert call(P, 0, 8, F32, 8, P, 8, 4, 1.0, P, None) == ARG
    assert call(P, 10, 8, F32, 0, P, 8, 4, 1.0, P, None) == ARG
    assert call(P, 10, 8, F32, 8, P, 8, 1 << 31, 1.0, P, None) == ARG
    assert call(P, 1 << 31, 8, F32, 8, P, 8, 4, 1.0, P, None) == ARG
    assert call(None, 10, 8, F32, 8, P, 8, 4, 1.0, P, None) == ARG
    assert call(None, 10, 8, F32, 8, None, 8, 0, 1.0, None, None) == OK
    back = lib.nerf_embedding_backward
    assert back(P, 7, 4, 8, P, 8, 10, 1.0, -1, P, P, None) == ARG
    assert back(P, F32, 4, 8, P, 1, 10, 1.0, -1, P, P, None) == ARG
    assert back(P, F32, 4, 8, P, 8, 10, 1.0, -1, None, P, None) == ARG
    assert back(P, F32, 4, 8, P, 8, 10, 1.0, -1, P, None, None) == ARG
    assert back(P, F32, 4, (1 << 20) + 1, P, 8, 10, 1.0, -1, P, P, None) == ARG
    assert lib.nerf_embedding_backward_workspace_bytes(4, 0, 8, F32) == -1
    assert lib.nerf_embedding_backward_workspace_bytes(0, 10, 8, F32) == 0
    # the sorted pairs and two partial rows per chunk
    assert lib.nerf_embedding_backward_workspace_bytes(100000, 70000, 32, F32) >= 8 * 100000


def test_dropout_entry_refuses():
    lib = _lib.load()
    call = lib.nerf_dropout
    assert call(P, None, 4, 10, 0.5, 1, None, 0, P, None) == ARG
    for p in (-0.1, 1.0000001, float("nan")):
        assert call(P, None, F32, 10, p, 1, None, 0, P, None) == ARG
    assert call(P, None, F32, 10, 0.5, 1, None, -1, P, None) == ARG
    assert call(P, None, F32, 10, 0.5, 1, None, (1 << 63) - 5, P, None) == ARG
    assert call(P, None, F32, -1, 0.5, 1, None, 0, P, None) == ARG
    assert call(None, None, F32, 10, 0.5, 1, None, 0, P, None) == ARG
    assert call(None, None, F32, 0, 0.5, 1, None, 0, None, None) == OK


def test_wrappers_refuse_cpu_tensors_and_foreign_types():
    x = torch.zeros(4, 8)
    ids = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ops.layernorm(x), lambda: ops.embedding(x, ids), lambda: ops.dropout(x, 0.5, 1),
                 lambda: ops.embedding_backward(x, ids, 10), lambda: ops.dropout_backward(x, 0.5, 1),
                 lambda: ops.layernorm_backward(x, x, None, x[:, 0], x[:, 0]),
                 lambda: layers.LayerNorm(8)(x), lambda: layers.Dropout(0.5)(x), lambda: layers.Embedding(4, 8)(ids)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    for call in (lambda: ops.layernorm([1.0]), lambda: ops.embedding(None, ids), lambda: ops.dropout(3, 0.5, 1)):
        with pytest.raises(ValueError, match="expected torch.Tensor"):
            call()
    with pytest.raises(ValueError):
        layers.Embedding(4, 8, padding_idx=4)
    with pytest.raises(ValueError):
        layers.Dropout(1.5)


def test_modules_share_their_state_with_torch():
    """Names and shapes of the parameters are torch.nn's: checkpoints go both ways."""
    for mine, theirs in ((layers.Embedding(7, 5), torch.nn.Embedding(7, 5)), (layers.LayerNorm(5), torch.nn.LayerNorm(5))):
        mine.load_state_dict(theirs.state_dict())
        theirs.load_state_dict(mine.state_dict())
        assert all(torch.equal(a, b) for a, b in zip(mine.parameters(), theirs.parameters()))
    assert float(layers.Embedding(7, 5, padding_idx=2).weight[2].detach().abs().sum()) == 0.0
    assert list(layers.LayerNorm(5, affine=False).parameters()) == [] and layers.LayerNorm(5, bias=False).bias is None
    x = torch.randn(3)
    assert layers.Dropout(0.5).eval()(x) is x and layers.Dropout(0.0)(x) is x


def test_functions_and_modules_refuse_before_the_backward_pass_would():
    """What training would refuse, or refuse only in the backward pass, is refused by the forward call and in evaluation."""
    table, ids = torch.zeros(4, 8, requires_grad=True), torch.zeros(4, dtype=torch.int64)
    for pad in (-1, 4):
        with pytest.raises(ValueError, match="padding_idx"):
            ops.EmbeddingFunction.apply(table, ids, 1.0, pad)
    x = torch.zeros(4, 8)
    drop = layers.Dropout(0.5).eval()
    for r in (x[:1], x.double(), x[0], 1.0):
        with pytest.raises(ValueError, match="residual"):
            drop(x, r)
    assert torch.equal(drop(x, x + 1), x + 1)


def test_dropout_modules_without_a_seed_have_one_each(monkeypatch):
    """Two modules of one seed would drop the same elements at every step.  The seeds repeat where a model is built again in
    the same order, whatever explicit seeds are in between, and an explicit one is taken as it is."""
    def build():
        monkeypatch.setattr(layers, "_unseeded", itertools.count())
        return [layers.Dropout(0.1).seed, layers.Dropout(0.1).seed, layers.Dropout(0.1, seed=3).seed, layers.Dropout().seed]
    seeds = build()
    assert len(set(seeds)) == 4 and seeds[2] == 3 and build() == seeds
    assert layers.Dropout(0.5, 0).seed == 0 and layers.Dropout(seed=2 ** 63).seed == 2 ** 63
