"""The device operators compute no gradients: a call that would cut a graph says so."""
import importlib
import warnings

import pytest


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def test_warns_only_where_a_graph_is_cut(jd, torch):
    dv = importlib.import_module("janus_doe_b200.devops")
    dv._lib()
    x = torch.zeros(3, requires_grad=True)
    with pytest.warns(UserWarning, match="some_op computes no gradients"):
        dv._forward_only("some_op", None, torch.zeros(2), x)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        dv._forward_only("some_op", None, x.detach())
        with torch.no_grad():
            dv._forward_only("some_op", x)


@pytest.mark.gpu
def test_every_operator_warns(jd, torch):
    i32 = dict(dtype=torch.int32, device="cuda")
    k, v = (torch.zeros((2, 16, 2, 64), device="cuda") for _ in range(2))
    kv = jd.PagedKV(k, v, torch.tensor([[0], [1]], **i32))
    x, seq = torch.randn((2, 2, 64), device="cuda"), torch.arange(2, **i32)
    lens, w = torch.ones(2, **i32), torch.ones(64, device="cuda")
    logits, cum, parent = torch.randn((2, 50), device="cuda"), torch.zeros(2, device="cuda"), torch.zeros((1, 2), **i32)

    def calls(g):
        def need(t):
            return t.clone().requires_grad_() if g else t
        yield lambda: jd.paged_append(kv, need(x), x, x, seq, seq * 0)
        yield lambda: jd.paged_append(kv, x, need(x), x, seq, seq * 0)
        yield lambda: jd.paged_append(kv, x, x, x, seq, seq * 0, q_norm=need(w), k_norm=w)
        yield lambda: jd.paged_attn(kv, need(x), lens, 1)
        yield lambda: jd.beam_select(need(logits), cum, 2, 2)
        yield lambda: jd.beam_reorder(parent, [(need(logits), torch.empty_like(logits))])

    for call in calls(True):
        with pytest.warns(UserWarning, match="computes no gradients"):
            call()
        with torch.no_grad(), warnings.catch_warnings():
            warnings.simplefilter("error")
            call()
    for call in calls(False):
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            call()
