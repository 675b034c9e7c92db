"""Copies of the paged caches, and objects that stand for one. On the CPU: the checks that ask for a device's tensors are
left out, everything else is the classes' own."""

from __future__ import annotations

import copy
import pickle

import pytest
import torch

from qwen35_hip import ops

PAGES, HEADS, PAGE, DIM = 3, 2, 16, 64


@pytest.fixture
def four(monkeypatch):
    monkeypatch.setattr(ops, "_checked", lambda dtype, *ts: None)
    return ops.kv4_cache(PAGES, HEADS, DIM, PAGE, device="cpu")


def pointers(cache, names):
    return tuple(getattr(cache, n).data_ptr() for n in names)


FOUR = ("k", "v", "k_scale", "k_min", "v_scale", "v_min")


def test_a_kv4_cache_changes_no_part(four):
    other = torch.zeros_like(four.k)
    for change in (lambda: four._replace(k=other), lambda: four._replace(args=four.args), lambda: four._replace(),
                   lambda: ops.Kv4Cache._make(four), lambda: ops.Kv4Cache._make([other] + list(four)[1:]),
                   lambda: setattr(four, "k", other), lambda: setattr(four, "more", 1), lambda: delattr(four, "k")):
        with pytest.raises((AttributeError, TypeError)):
            change()
    assert four.args[:6] == pointers(four, FOUR)


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c))])
def test_a_copy_of_a_kv4_cache_has_its_own_tensors_pointers(four, how):
    four.k.fill_(7)
    c = how(four)
    assert type(c) is ops.Kv4Cache
    assert c.args[:6] == pointers(c, FOUR) and c.args[6:] == four.args[6:] == (PAGES, PAGE, HEADS, DIM)
    assert (c.pages, c.page, c.heads, c.dim) == (PAGES, PAGE, HEADS, DIM) and bool((c.k == 7).all())
    assert (c.k.data_ptr() == four.k.data_ptr()) == (how is copy.copy)


EIGHT = ("k", "v", "k_scale", "v_scale")


@pytest.fixture
def eight(monkeypatch):
    monkeypatch.setattr(ops, "_checked", lambda dtype, *ts: None)
    return ops.kv8_cache(PAGES, HEADS, DIM, PAGE, device="cpu")


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c))])
def test_a_copy_of_a_kv8_cache_has_its_own_tensors_pointers(eight, how):
    eight.k.fill_(7)
    c = how(eight)
    assert type(c) is ops.Kv8Cache
    assert c.args == pointers(c, EIGHT) + (PAGES, PAGE, HEADS, DIM) and bool((c.k == 7).all())
    assert (c.k.data_ptr() == eight.k.data_ptr()) == (how is copy.copy)
    with pytest.raises(AttributeError):
        c.k = eight.k


class Lookalike:
    """A program's own object with a Kv8Cache's fields."""

    def __init__(self, cache):
        for name in ops.Kv8Cache.__slots__:
            setattr(self, name, getattr(cache, name))


def test_the_8_bit_calls_take_any_object_with_a_caches_fields(eight, four):
    """They refuse a 4-bit cache, which has other arrays behind its pointers, and nothing else by its type: what these calls
    refuse here are the tensors, which are not a device's."""
    x, i = torch.zeros((1, HEADS, DIM)), torch.zeros(1, dtype=torch.int32)

    def calls(c):
        return (lambda: ops.kv8_store_rows(x, x, i, c), lambda: ops.attn_kv8_rows(x, c, i.view(1, 1), i, i))
    for call in calls(Lookalike(eight)):
        with pytest.raises(ValueError) as e:
            call()
        assert "expected a Kv" not in str(e.value)
    for call in (*calls(four), lambda: ops.kv8_read_rows(four, i)):
        with pytest.raises(ValueError, match="expected a Kv8Cache, got Kv4Cache"):
            call()
    for call in (lambda: ops.kv4_store_rows(x, x, i, eight), lambda: ops.kv4_read_rows(eight, i),
                 lambda: ops.attn_kv4_rows(x, eight, i.view(1, 1), i, i)):
        with pytest.raises(ValueError, match="expected a Kv4Cache, got Kv8Cache"):
            call()
