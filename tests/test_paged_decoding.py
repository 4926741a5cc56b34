"""Where the paged caches and the token log probabilities are used: the decoder's paged self-attention cache under the beam search, the search
that ranks only the likeliest symbols, and the cross entropy with an entropy term.  Host logic over the float64 restatement of the kernels'
contracts; the same calls on the device are in test_gpu_paged_decoding.py."""
import contextlib
import gc
import weakref

import pytest
import torch

from neurst_amd.layers.attentions.paged_kv_cache import PagedKVCache
from neurst_amd.layers.search.beam_search import sequence_beam_search
from oracle import kernel_emulation as E


@pytest.fixture
def cpu_kernels(monkeypatch):
    return E.install(monkeypatch)


def _toy_model(device="cpu", dtype="float32", V=20, seed=5):
    from neurst_amd.models import build_model
    from neurst_amd.utils.hparams_sets import get_hyper_parameters
    return build_model(get_hyper_parameters("speech_transformer_toy"), {"audio_feature_dim": 16, "audio_feature_channels": 1},
                       {"vocab_size": V, "eos_id": V - 1, "bos_id": V - 2, "unk_id": V - 3}, device=device, dtype=dtype, seed=seed)


def _inputs(B=2, T=36, seed=8):
    g = torch.Generator().manual_seed(seed)
    return {"src": torch.randn(B, T, 16, 1, generator=g), "src_length": torch.tensor([T] + [T - 11] * (B - 1))}


@pytest.mark.parametrize("page_size", [1, 3, 4, 64])
@pytest.mark.parametrize("beam,top_k", [(1, 1), (3, 2), (4, 1)])
def test_beam_search_over_pages_equals_the_dense_cache(cpu_kernels, page_size, beam, top_k):
    from neurst_amd.layers.search import BeamSearch
    model, inputs = _toy_model(seed=11), _inputs()
    kw = dict(beam_size=beam, top_k=top_k, maximum_decode_length=8)
    h0, s0 = BeamSearch(**kw)(model, inputs)
    h1, s1 = BeamSearch(page_size=page_size, **kw)(model, inputs)
    assert torch.equal(h0, h1) and torch.allclose(s0, s1, atol=1e-6)
    h2, s2 = BeamSearch(page_size=page_size, fused_scores=True, **kw)(model, inputs)
    assert torch.equal(h0, h2) and torch.allclose(s0, s2, atol=1e-5)


def test_paged_steps_equal_dense_steps_and_a_full_cache_is_an_error(cpu_kernels):
    model, inputs = _toy_model(), _inputs(B=3)
    ids = torch.randint(0, 17, (3, 6), generator=torch.Generator().manual_seed(1))
    fd, init_d, _ = model.get_symbols_to_logits_fn(inputs, beam_size=1, decode_padded_length=6)
    fp, init_p, _ = model.get_symbols_to_logits_fn(inputs, beam_size=1, decode_padded_length=6, page_size=4)
    cache = init_p["decoder_internal_cache"]
    for t in range(6):
        assert torch.allclose(fd(ids[:, t], init_d["decoder_internal_cache"], t), fp(ids[:, t], cache, t), atol=1e-6)
    assert all(st["self_attention"]["len"] == 6 for st in cache["decoding_states"].values()) and cache["paged"].len == 6
    with pytest.raises(RuntimeError, match="6 positions is full"):
        fp(ids[:, 0], cache, 6)


def test_paged_cache_of_rows_with_different_lengths(cpu_kernels):
    cache = PagedKVCache(2, 4, 2, 8, max_length=10, page_size=3, dtype=torch.float32, device="cpu")
    g = torch.Generator().manual_seed(0)
    hist = [[] for _ in range(4)]
    for new in ([3, 0, 5, 1], [1, 1, 1, 1], [0, 2, 0, 1]):
        cache.extend(torch.tensor(new, dtype=torch.int32), longest=max(new), max_tokens=sum(new))
        rows = torch.randn(sum(new), 2, 2, 2, 8, generator=g)               # [token, layer, k|v, head, dh]
        at = 0
        for r, n in enumerate(new):
            hist[r] += [rows[at + i] for i in range(n)]
            at += n
        for layer in range(2):
            cache.append(layer, rows[:, layer, 0], rows[:, layer, 1])
        q = torch.randn(4, 2, 8, generator=g)
        for layer in range(2):
            out = cache.attend(layer, q)
            for r in range(4):
                if not hist[r]:
                    assert float(out[r].abs().max()) == 0.0
                    continue
                k, v = (torch.stack([h[layer, i] for h in hist[r]]).double() for i in range(2))
                p = torch.softmax(torch.einsum("thd,hd->ht", k, q[r].double()) / 8 ** 0.5, -1)
                assert torch.allclose(out[r].double(), torch.einsum("ht,thd->hd", p, v), atol=1e-6)
    with pytest.raises(RuntimeError, match="full"):
        cache.extend(torch.full((4,), 3, dtype=torch.int32), longest=3)
    with pytest.raises(ValueError, match="at least one token"):
        PagedKVCache(1, 1, 1, 8, 4, 0, torch.float32, "cpu")
    with pytest.raises(ValueError, match="up to 256"):
        PagedKVCache(1, 1, 1, 300, 4, 2, torch.float32, "cpu")


def run_rows_that_grow_in_turn(device, tol):
    """Prompts that arrive one after the other, each for another row: a row is full when IT is, not when the prompts together are as long."""
    rows, heads, dh, longest = 4, 2, 8, 6
    cache = PagedKVCache(1, rows, heads, dh, max_length=longest, page_size=4, dtype=torch.float32, device=device)
    g = torch.Generator().manual_seed(2)
    hist = [torch.zeros(0, 2, heads, dh) for _ in range(rows)]
    for new, length in (([5, 0, 0, 0], 5), ([0, 5, 0, 0], 5), ([0, 0, 6, 0], 6), ([1, 0, 0, 3], 6)):
        kv = torch.randn(sum(new), 2, heads, dh, generator=g)
        cache.extend(torch.tensor(new, dtype=torch.int32, device=device), longest=max(new), max_tokens=sum(new), length=length)
        assert cache.len == length
        cache.append(0, kv[:, 0].to(device), kv[:, 1].to(device))
        hist = [torch.cat([h, part]) for h, part in zip(hist, kv.split(new))]
        q = torch.randn(rows, heads, dh, generator=g)
        out = cache.attend(0, q.to(device)).cpu().double()
        assert cache.seq_lens.tolist() == [h.shape[0] for h in hist]
        for r in range(rows):
            k, v = hist[r][:, 0].double(), hist[r][:, 1].double()
            want = torch.einsum("ht,thd->hd", torch.softmax(torch.einsum("thd,hd->ht", k, q[r].double()) / dh ** 0.5, -1), v)
            assert float((out[r] - want).abs().max()) <= tol, (new, r)
    state = cache.table.clone(), cache.seq_lens.clone(), cache.cursor.clone()
    with pytest.raises(RuntimeError, match="6 positions is full"):
        cache.extend(torch.tensor([0, 2, 0, 0], dtype=torch.int32, device=device), longest=2, length=7)
    with pytest.raises(RuntimeError, match="6 positions is full"):            # the host does not know: the longest row might be the one
        cache.extend(torch.tensor([0, 1, 0, 0], dtype=torch.int32, device=device))
    with pytest.raises(ValueError, match="at most -1"):
        cache.extend(length=-1)
    assert all(torch.equal(a, b) for a, b in zip(state, (cache.table, cache.seq_lens, cache.cursor))) and cache.len == 6
    cache.extend(torch.tensor([0, 1, 0, 3], dtype=torch.int32, device=device), longest=3, max_tokens=4, length=6)
    assert cache.seq_lens.tolist() == [6, 6, 6, 6]


def test_rows_that_grow_in_turn(cpu_kernels):
    run_rows_that_grow_in_turn("cpu", 1e-6)


@pytest.mark.parametrize("beam,top_k,alpha,min_len,enable_unk", [(1, 1, 0.6, 0, False), (4, 4, 1.0, 0, False), (3, 2, -1.0, 0, True),
                                                                 (5, 3, 0.0, 6, False), (4, 2, 0.6, 11, False)])
def test_search_over_the_likeliest_symbols_equals_the_full_search(cpu_kernels, beam, top_k, alpha, min_len, enable_unk):
    from test_search import _ToyLM
    vocab, batch, bos, eos, unk = 17, 3, 15, 16, 14
    kw = dict(beam_size=beam, top_k=top_k, length_penalty=alpha, extra_decode_length=4, maximum_decode_length=12,
              minimum_decode_length=min_len, enable_unk=enable_unk)
    got = []
    for fused in (False, True):
        lm = _ToyLM(vocab, batch, seed=beam * 10 + top_k, eos_boost=0.4)
        fn, reorder = lm.step_fn(beam, eos)
        init = {"decoder_input": torch.full((batch,), bos), "encoder_inputs_maxlen": 5, "eos_id": eos, "unk_id": unk,
                "decoder_internal_cache": {"state": torch.zeros(batch * beam, dtype=torch.int64)}}
        got.append(sequence_beam_search(fn, init, reorder_cache_fn=reorder, fused_scores=fused, **kw))
    assert torch.equal(got[0][0], got[1][0]) and torch.allclose(got[0][1], got[1][1], rtol=1e-5, atol=1e-5)


def test_search_falls_back_where_the_vocabulary_is_smaller_than_the_expansion(cpu_kernels):
    """beam + masked symbols > vocabulary: the full ranking takes over (and the kernel is not asked for more symbols than there are)."""
    table = torch.randn(4, 4, generator=torch.Generator().manual_seed(1))
    init = {"decoder_input": torch.tensor([2]), "decoder_internal_cache": {}, "encoder_inputs_maxlen": 3, "eos_id": 3, "unk_id": 0}
    kw = dict(beam_size=4, top_k=2, maximum_decode_length=5)
    a = sequence_beam_search(lambda ids, c, t: table[ids], init, **kw)
    b = sequence_beam_search(lambda ids, c, t: table[ids], init, fused_scores=True, **kw)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------------------------------------ criterion
def entropy_loss_reference(logits, trg, weights, beta):
    lp = torch.log_softmax(logits.double(), -1)
    nll = -lp.gather(-1, trg[..., None])[..., 0]
    H = -(lp.exp() * lp).sum(-1)
    return ((nll - beta * H) * weights.double()).sum() / weights.double().sum()


@pytest.mark.parametrize("beta", [0.0, 0.3])
def test_entropy_regularized_cross_entropy(cpu_kernels, beta):
    from neurst_amd.criterions import build_criterion
    g = torch.Generator().manual_seed(0)
    B, L, V = 3, 5, 11
    logits = torch.randn(B, L, V, generator=g).double().requires_grad_()
    trg, length = torch.randint(0, V, (B, L), generator=g), torch.tensor([5, 3, 1])
    inp = {"trg": trg, "trg_length": length}
    weights = (torch.arange(L)[None, :] < length[:, None]).double()
    want = entropy_loss_reference(logits, trg, weights, beta)
    want.backward()
    crit = build_criterion({"criterion.class": "entropy_regularized_cross_entropy", "criterion.params": {"entropy_weight": beta}})
    loss = crit.reduce_loss(inp, logits.detach().float())
    want = want.detach()
    assert abs(float(loss) - float(want)) < 1e-6
    grad = crit.backward(loss_scale=2.0, loss_scale_dev=torch.tensor([0.5]))
    assert float((grad.double() - logits.grad).abs().max()) < 1e-7
    nll, n, tokens = crit(inp, logits.detach().float())
    assert tokens.tolist() == [5, 3, 1] and float(n) == 3 and abs(float(nll.sum() / tokens.sum()) - float(want)) < 1e-6
    if beta == 0.0:
        plain = build_criterion({"criterion.class": "label_smoothed_cross_entropy", "criterion.params": {}})
        assert abs(float(plain.reduce_loss(inp, logits.detach().float())) - float(loss)) < 1e-6
        assert float((plain.backward() - grad).abs().max()) < 1e-7


def run_entropy_training(device, dtype, tol):
    """A training step with the criterion: the parameters' gradients equal those of the formula's d(logits), handed to the same backward pass."""
    from neurst_amd.criterions import build_criterion
    from neurst_amd.models import build_model
    from neurst_amd.optimizers import build_optimizer
    from neurst_amd.training.train_step import TrainStep
    from neurst_amd.utils.hparams_sets import get_hyper_parameters
    hp = get_hyper_parameters("speech_transformer_toy")
    for k in list(hp["model.params"]):
        if k.endswith("dropout_rate"):
            hp["model.params"][k] = 0.0
    model = build_model(hp, {"audio_feature_dim": 16, "audio_feature_channels": 1}, {"vocab_size": 20, "eos_id": 19, "bos_id": 18, "unk_id": 17},
                        device=device, dtype=dtype, seed=5)
    inputs = dict(_inputs(), trg=torch.tensor([[3, 4, 19], [5, 19, 19]]), trg_length=torch.tensor([3, 2]),
                  trg_input=torch.tensor([[18, 3, 4], [18, 5, 19]]))
    inputs = {k: v.to(device) for k, v in inputs.items()}
    crit = build_criterion({"criterion.class": "EntropyRegularizedCrossEntropy", "criterion.params": {"entropy_weight": 0.2}})
    logits = model(inputs, is_training=True)
    leaf = logits.detach().cpu().double().requires_grad_()
    weights = (torch.arange(3)[None, :] < inputs["trg_length"].cpu()[:, None]).double()
    want = entropy_loss_reference(leaf, inputs["trg"].cpu(), weights, 0.2)
    want.backward()
    model.backward(leaf.grad.to(logits.dtype).to(logits.device))
    ref = model.store.grad.clone()
    logits = model(inputs, is_training=True)
    loss = crit.reduce_loss(inputs, logits)
    assert abs(float(loss) - want.item()) <= tol * abs(want.item())
    model.backward(crit.backward())
    assert float((model.store.grad - ref).norm()) <= tol * float(ref.norm())
    opt = build_optimizer({"optimizer.class": "Adam", "optimizer.params": {"learning_rate": 1e-3}}).bind(model.store)
    before = model.store.master.clone()
    assert torch.isfinite(TrainStep(model, crit, opt)(inputs)) and not torch.equal(before, model.store.master)


def test_entropy_regularized_training_of_the_model(cpu_kernels):
    # f32 results of float64 arithmetic on both sides: the two d(logits) differ by a rounding (2^-24) each, carried linearly
    run_entropy_training("cpu", "float32", 1e-5)


# ------------------------------------------------------------------------------------------------ captured decoding steps
class _GraphStub(object):
    """In the place of a HIP graph: capturing runs the step once, replaying does nothing (what the first batch of a session needs)."""
    collector_on = []

    def __init__(self):
        self.in_cycle = self                                     # like everything that waits for the cyclic collector

    def pool(self):
        return 1

    def replay(self):
        pass


@contextlib.contextmanager
def _capture_stub(graph, pool=None, **kwargs):
    _GraphStub.collector_on.append(gc.isenabled())
    yield


@pytest.fixture
def stubbed_graphs(cpu_kernels, monkeypatch):
    monkeypatch.setattr(torch.cuda, "CUDAGraph", _GraphStub)
    monkeypatch.setattr(torch.cuda, "graph", _capture_stub)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    _GraphStub.collector_on = []
    return _GraphStub


@pytest.mark.parametrize("page_size", [None, 4])
def test_no_collection_runs_while_a_decoding_step_is_captured(stubbed_graphs, monkeypatch, page_size):
    """A collection in the middle of a capture may destroy the captured graphs of a model that was dropped earlier: the process would end.
    What is there to collect goes before the capture, and the collector comes back behind it, also behind one that fails."""
    from neurst_amd.layers.search import BeamSearch
    model, inputs = _toy_model(seed=11), _inputs()
    kw = dict(beam_size=3, top_k=2, maximum_decode_length=8, page_size=page_size)
    h0, s0 = BeamSearch(**kw)(model, inputs)
    garbage = weakref.ref(stubbed_graphs())                      # freed by the cyclic collector alone
    assert gc.isenabled() and garbage() is not None
    h1, s1 = BeamSearch(use_graphs=True, **kw)(model, inputs)
    assert torch.equal(h0, h1) and torch.equal(s0, s1)
    assert stubbed_graphs.collector_on and not any(stubbed_graphs.collector_on) and gc.isenabled() and garbage() is None

    def failing(graph, pool=None):
        raise RuntimeError("no capture")
    monkeypatch.setattr(torch.cuda, "graph", failing)
    with pytest.raises(RuntimeError, match="no capture"):
        BeamSearch(use_graphs=True, **dict(kw, maximum_decode_length=7))(model, inputs)
    assert gc.isenabled()
    gc.disable()
    try:                                                         # off before: off afterwards
        monkeypatch.setattr(torch.cuda, "graph", _capture_stub)
        BeamSearch(use_graphs=True, **dict(kw, maximum_decode_length=6))(model, inputs)
        assert not gc.isenabled()
    finally:
        gc.enable()


@pytest.mark.parametrize("page_size", [None, 4])
def test_a_dropped_model_takes_its_captured_steps_along(stubbed_graphs, page_size):
    """... at once, not when the cyclic collector comes by; and the step function alone keeps its model alive."""
    model, inputs = _toy_model(seed=11), _inputs()
    fn, init, _ = model.get_symbols_to_logits_fn(inputs, beam_size=2, decode_padded_length=6, use_graphs=True,
                                                 **({"page_size": page_size} if page_size else {}))
    alive = weakref.ref(model)
    session = weakref.ref(next(iter(model._decode_sessions.values())))
    del model
    logits = fn(torch.full((4,), 18), init["decoder_internal_cache"], 0)
    assert logits.shape == (4, 20) and alive() is not None and len(session().graphs) == 1
    gc.disable()
    try:
        del fn, init
        assert alive() is None and session() is None
    finally:
        gc.enable()
