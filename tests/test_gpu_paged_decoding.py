"""Paged beam search and the entropy-regularised criterion on the device (the host logic is in test_paged_decoding.py)."""
import pytest
import torch

from test_paged_decoding import _inputs, _toy_model, run_entropy_training, run_rows_that_grow_in_turn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _dev_inputs(**kw):
    return {k: v.to(DEV) for k, v in _inputs(**kw).items()}


@pytest.mark.parametrize("page_size", [3, 16])
@pytest.mark.parametrize("beam,top_k", [(1, 1), (4, 2)])
def test_paged_beam_search_equals_the_dense_one_in_float32(page_size, beam, top_k):
    """float32 attention differs by the order of its sums only (1e-6 of the logits): the hypotheses of the toy model, whose candidates lie
    1e-3 apart and more, are the same."""
    from neurst_amd.layers.search import BeamSearch
    model, inputs = _toy_model(DEV, "float32", seed=11), _dev_inputs()
    kw = dict(beam_size=beam, top_k=top_k, maximum_decode_length=9)
    h0, s0 = BeamSearch(**kw)(model, inputs)
    for extra in (dict(), dict(fused_scores=True)):
        h1, s1 = BeamSearch(page_size=page_size, **kw, **extra)(model, inputs)
        assert torch.equal(h0, h1) and torch.allclose(s0, s1, atol=1e-4), extra
    h2, s2 = BeamSearch(fused_scores=True, **kw)(model, inputs)
    assert torch.equal(h0, h2) and torch.allclose(s0, s2, atol=1e-4)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_paged_steps_follow_the_full_forward(dtype):
    V, B, L = 20, 3, 7
    model, inputs = _toy_model(DEV, dtype), _dev_inputs(B=3)
    g = torch.Generator().manual_seed(3)
    trg_input = torch.cat([torch.full((B, 1), V - 2), torch.randint(0, V - 3, (B, L - 1), generator=g)], 1).to(DEV)
    full = model(dict(inputs, trg_input=trg_input), is_training=False).float()
    fn, init, _ = model.get_symbols_to_logits_fn(inputs, beam_size=1, decode_padded_length=L, page_size=4)
    # the tolerances of the dense decoding test: five times the relative bound of one kernel (1e-3 / 1e-2)
    tol = 5 * (1e-3 if dtype == "float32" else 1e-2) * float(full.abs().max())
    for t in range(L):
        step = fn(trg_input[:, t], init["decoder_internal_cache"], t).float()
        assert float((step - full[:, t]).abs().max()) <= tol, t


@pytest.mark.parametrize("fused", [False, True])
def test_graph_replayed_paged_decoding_equals_eager_paged_decoding(fused):
    """Captured steps over the static paged cache, for a second and a third batch that replay the first one's graphs."""
    from neurst_amd.layers.search import BeamSearch
    model = _toy_model(DEV, "bfloat16", seed=21)
    kw = dict(beam_size=3, top_k=2, maximum_decode_length=9, page_size=4, fused_scores=fused)
    eager, graphed = BeamSearch(**kw), BeamSearch(use_graphs=True, **kw)
    for seed in (1, 2, 3, 1):
        inputs = _dev_inputs(B=3, T=44, seed=seed)
        h0, s0 = eager(model, inputs)
        h1, s1 = graphed(model, inputs)
        assert torch.equal(h0, h1) and torch.equal(s0, s1), seed
    dense = BeamSearch(beam_size=3, top_k=2, maximum_decode_length=9, use_graphs=True)
    assert dense(model, inputs)[0].shape == h0.shape and len(model._decode_sessions) == 2      # sessions of their own


def test_rows_that_grow_in_turn():
    """float32, 6 tokens, heads of 8: a score of size 10 is off by (8 + 7) 2^-24 of it, the weights by twice that, the sums by 28 2^-24 -- 2e-5
    of values of size 4."""
    run_rows_that_grow_in_turn(DEV, 8e-5)


@pytest.mark.parametrize("dtype,tol", [("float32", 1e-5), ("bfloat16", 2.0 ** -6)])
def test_entropy_regularized_training_step(dtype, tol):
    """float32: the kernels' d(logits) is within 1e-6 of the formula's.  bf16: both sides round d(logits) to bf16 (2^-8 each at most), from
    statistics that agree to 1e-6; the rest of the backward pass is the same linear map with the same roundings of other values
    (another 2^-8 on each side)."""
    run_entropy_training(DEV, dtype, tol)


def test_entropy_regularized_training_replays_from_a_graph():
    """Graph replay equals eager steps with this criterion too (float32, no dropout: the embedding gradient's atomics leave last-bit
    differences, 1e-5 as in the test of the label-smoothed criterion)."""
    from test_gpu_graph import _batch, _setup
    from neurst_amd.criterions import build_criterion
    batches, res = [_batch(300 + i) for i in range(5)], {}
    for use_graph in (False, True):
        model, step, _ = _setup("float32", 0.0, use_graph)
        step.criterion = build_criterion({"criterion.class": "entropy_regularized_cross_entropy", "criterion.params": {"entropy_weight": 0.1}})
        losses = []
        for b in batches:
            losses.append(float(step(b)))
            torch.cuda.synchronize()
        res[use_graph] = losses
        assert step.replays == (len(batches) - 1 if use_graph else 0)
    for a, b in zip(res[False], res[True]):
        assert abs(a - b) <= 1e-5 * max(1.0, abs(a)), res
