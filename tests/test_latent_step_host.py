"""Host-side behaviour of ``latent.mla_step`` and ``LatentCache`` (no GPU needed)."""

from __future__ import annotations

import copy
import types

import pytest
import torch

from conftest import pkg


def _step_args(DR=0, grad=False):
    mod = types.SimpleNamespace(
        num_heads=2, qk_nope_head_dim=8, qk_rope_head_dim=DR, v_head_dim=8, scale=0.1,
        kv_b_proj=torch.nn.Linear(128, 32, bias=False), o_proj=torch.nn.Linear(16, 4, bias=False))
    state = {"cache": pkg().LatentCache(2, 16, 128, device="cpu"),
             "block_table": torch.zeros(2, 1, dtype=torch.int32),
             "lens": torch.tensor([3, 5], dtype=torch.int32)}
    x, q = torch.zeros(2, 1, 4), torch.zeros(2, 1, 2, 8)
    return [mod, x, q, None, torch.zeros(2, 1, 128, requires_grad=grad), None, state]


@pytest.mark.parametrize("spoil", ["cpu", "grad", "width", "rope", "weight"])
def test_a_refused_step_leaves_the_lengths_alone(spoil):
    """A refusal of ``mla_step`` comes before the caller's lengths change, or takes the
    change back: a second try finds what the first one found."""
    args = _step_args(DR=64 if spoil == "rope" else 0, grad=spoil == "grad")
    if spoil == "width":
        args[4] = torch.zeros(2, 1, 64)
    if spoil == "weight":
        args[0].kv_b_proj = torch.nn.Linear(64, 32, bias=False)
    for _ in range(2):
        with pytest.raises((RuntimeError, TypeError)):
            pkg().latent.mla_step(*args, True)
        assert args[6]["lens"].tolist() == [3, 5]


def test_the_pool_of_a_cache_is_fixed():
    """The kernels' argument block holds the pool's addresses and sizes, so none of them can
    be replaced behind it; a larger pool is another cache."""
    kb = pkg()
    c = kb.LatentCache(2, 16, 128, 64, device="cpu")
    other = kb.LatentCache(4, 16, 128, 64, device="cpu")
    for name in ("codes", "scales", "rope", "dtype", "device", "num_pages", "page_size",
                 "kv_lora_rank", "rope_dim"):
        before = getattr(c, name)
        with pytest.raises(AttributeError, match="from_tensors"):
            setattr(c, name, getattr(other, name))
        with pytest.raises(AttributeError, match="from_tensors"):
            delattr(c, name)
        assert getattr(c, name) is before
    grown = kb.LatentCache.from_tensors(other.codes, other.scales, other.rope)
    assert grown.num_pages == 4 and grown.codes is other.codes


def test_a_copied_cache_has_its_own_addresses():
    kb = pkg()
    c = kb.LatentCache(2, 16, 128, 64, device="cpu")
    for other, own in ((copy.deepcopy(c), True), (copy.copy(c), False)):
        a = kb._lib.MlaCacheArgs.from_buffer_copy(other._args)
        assert (a.codes, a.scales, a.rope) == tuple(t.data_ptr() for t in (other.codes, other.scales, other.rope))
        assert (other.codes.data_ptr() != c.codes.data_ptr()) == own and other.dtype is c.dtype
