"""predict_cached: it scores the tokens that user_offsets name, for the sequences that are named, and
leaves the cache as it was where it raises.  Its scores are those of the model's parts called one
after the other, bit for bit; each layer's attention is held to the 64-bit form elsewhere."""
import pytest
import torch

pytestmark = pytest.mark.gpu

LENS = [40, 100, 17]


@pytest.fixture(scope="module")
def setting(cuda_device):
    from cti_b200 import synth
    from cti_b200.model import build_ctr_model

    bb = synth.bag_batch(batch=sum(LENS) + 20, seed=4, vocab_hi=2e4)
    model = build_ctr_model(bb.vocab.tolist(), num_layers=2, num_experts=8, dim_ff=256)
    synth.init_ctr_model(model)
    with torch.no_grad():
        model.rep_encoder.emb.weight = torch.nn.Parameter(
            synth.embedding_table(bb.total_rows, 64, seed=1), requires_grad=False)
        # Larger weights than a model starts with: histories matter.
        for layer in model.seq_encoder.qkv_proj:
            layer.weight.mul_(8)
    model.to(cuda_device).prepare_for_inference()
    return model, bb


def _batch(bb, ranges, user_offsets):
    """The flat layout of some token ranges."""
    offs = bb.row_offsets.view(bb.features, -1)
    vals, ro, vo, start = [], [], [], 0
    for f in range(bb.features):
        base = int(bb.val_offsets[f])
        pieces = [bb.values[base + int(offs[f, a]):base + int(offs[f, b])] for a, b in ranges]
        counts = torch.cat([offs[f, a + 1:b + 1] - offs[f, a:b] for a, b in ranges])
        ro.append(torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(counts, 0)]))
        vals.append(torch.cat(pieces))
        vo.append(start)
        start += vals[-1].numel()
    return {"_flat_values": torch.cat(vals), "_flat_row_offsets": torch.cat(ro),
            "_val_offsets": torch.tensor(vo), "user_offsets": torch.tensor(user_offsets)}


def _cache(model, **kw):
    return model.sequence_cache(**{**dict(max_seqs=8, num_pages=10, max_tokens=256), **kw})


def _histories(model, bb, cache):
    """Sequences 5, 0 and 7 with LENS tokens."""
    cu = [0, 40, 140, 157]
    return model.predict_cached(_batch(bb, [(0, 157)], cu), cache, [5, 0, 7])


def _state(c):
    return (c.free_pages, [c.length(i) for i in range(c.max_seqs)])


def _by_parts(model, batch, cache, seqs, new):
    x = model.rep_encoder(batch)
    h, _ = model.seq_encoder(x[:sum(new)], cache.extend(seqs, new))
    return model.head(h, want_logits=False)[1]


def test_scores_are_the_parts_and_depend_on_the_history(setting):
    from cti_b200 import _lib

    model, bb = setting
    a, b = _cache(model), _cache(model)
    first = _histories(model, bb, a)
    assert torch.equal(first, _by_parts(model, _batch(bb, [(0, 157)], [0]), b, [5, 0, 7], LENS))
    batch = _batch(bb, [(157, 163)], [0, 1, 4, 6])
    second = model.predict_cached(batch, a, [7, 5, 0])
    assert torch.equal(second, _by_parts(model, batch, b, [7, 5, 0], [1, 3, 2]))
    assert [a.length(s) for s in (5, 0, 7)] == [43, 102, 18]
    # Other histories, or none, give other scores, for every token.
    none = model.predict_cached(batch, _cache(model), [7, 5, 0])
    c = _cache(model)
    _histories(model, bb, c)
    other = model.predict_cached(batch, c, [0, 7, 5])
    _lib.raise_on_status(second.device)
    assert torch.isfinite(second).all()
    assert (second != none).all() and (second != other).all()


def test_offsets_that_do_not_start_at_the_first_token(setting):
    """Tokens before, and behind, belong to no sequence: they are not scored."""
    model, bb = setting
    a, b = _cache(model), _cache(model)
    for c in (a, b):
        _histories(model, bb, c)
    want = model.predict_cached(_batch(bb, [(159, 164)], [0, 1, 3, 5]), a, [7, 5, 0])
    got = model.predict_cached(_batch(bb, [(157, 167)], [2, 3, 5, 7]), b, [7, 5, 0])
    assert got.shape == (10,) and torch.equal(got[2:7], want)
    assert torch.isnan(got[:2]).all() and torch.isnan(got[7:]).all()
    assert _state(a) == _state(b)
    # ... and the keys and values are those tokens'.
    batch = _batch(bb, [(170, 172)], [0, 1, 2])
    assert torch.equal(model.predict_cached(batch, a, [5, 0]), model.predict_cached(batch, b, [5, 0]))


def test_a_forward_that_raises_leaves_the_cache_as_it_was(setting, monkeypatch):
    model, bb = setting
    a, b = _cache(model), _cache(model)
    for c in (a, b):
        _histories(model, bb, c)
    state = _state(a)
    batch = _batch(bb, [(157, 177)], [0, 19, 20])
    for where in ("seq_encoder.moe.1", "seq_encoder.out_proj.0", "rep_encoder"):
        module = model.get_submodule(where)

        def fails(*args, **kw):
            raise RuntimeError("out of memory")

        monkeypatch.setattr(module, "forward", fails)
        with pytest.raises(RuntimeError, match="out of memory"):
            model.predict_cached(batch, a, [0, 5])
        monkeypatch.undo()
        assert _state(a) == state
    monkeypatch.setattr(model, "head", fails)
    with pytest.raises(RuntimeError):
        model.predict_cached(batch, a, [0, 5])
    monkeypatch.undo()
    assert _state(a) == state
    want = model.predict_cached(batch, b, [0, 5])
    assert torch.equal(model.predict_cached(batch, a, [0, 5]), want)
    assert _state(a) == _state(b) != state


def test_wrong_calls_are_refused_and_change_nothing(setting):
    import cti_b200

    model, bb = setting
    enc, dev = model.seq_encoder, model.linear[0].weight.device
    c = _cache(model)
    _histories(model, bb, c)
    state = _state(c)
    for offsets, seqs, error in (([0, 1, 7], [5, 0], ValueError),   # past the batch's tokens
                                 ([0, 3, 2], [5, 0], ValueError), ([0, 3, 0], [5, 0], ValueError),
                                 ([-1, 1, 2], [5, 0], ValueError), ([0, 6], [5, 0], ValueError),
                                 ([0, 3, 6], [5, 5], ValueError), ([0, 0, 0], [5, 9], IndexError),
                                 ([0, 3, 6], [5, 8], IndexError)):
        with pytest.raises(error):
            model.predict_cached(_batch(bb, [(157, 163)], offsets), c, seqs)
        assert _state(c) == state
    batch = _batch(bb, [(157, 163)], [0, 3, 6])
    args = dict(num_layers=enc.num_layers, max_seqs=8, num_pages=10, kv_heads=enc.n_heads,
                head_dim=enc.head_dim, max_tokens=256, device=dev)
    for kw in (dict(num_layers=enc.num_layers + 1), dict(kv_heads=2 * enc.n_heads),
               dict(kv_heads=max(1, enc.n_heads // 2)), dict(head_dim=128 if enc.head_dim < 128 else 64),
               dict(dtype=torch.float16), dict(device="cpu")):
        other = cti_b200.SequenceCache(**{**args, **kw})
        with pytest.raises(ValueError):
            model.predict_cached(batch, other, [5, 0])
        assert _state(other) == (10, [0] * 8)
    e = c.extend([5], [3])
    with pytest.raises(ValueError):  # fewer tokens than the extension holds
        enc(torch.zeros(2, enc.d_model, dtype=torch.bfloat16, device=dev), e)
    c.undo(e)
    assert _state(c) == state
    assert model.predict_cached(_batch(bb, [(157, 163)], [0, 0, 0]), c, [5, 0]).shape == (6,)
    assert _state(c) == state


def test_extend_is_refused_inside_a_capture(setting):
    """Its book-keeping would happen once, for every replay; the forward itself can be captured, with
    the extension's tensors as its inputs."""
    from cti_b200 import _lib

    model, bb = setting
    c = _cache(model)
    _histories(model, bb, c)
    state = _state(c)
    enc, dev = model.seq_encoder, c.device
    x = torch.randn(4, enc.d_model, device=dev).bfloat16()
    e = c.extend([5, 0], [1, 3])
    want, _ = enc(x, e)  # warm-up too; the tokens are appended anew by each run, to their places
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(RuntimeError, match="captured"):
            c.extend([7], [1])
        got, _ = enc(x, e)
    for _ in range(2):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize(dev)
        assert torch.equal(got, want)
    _lib.raise_on_status(dev)
    assert c.length(7) == state[1][7] and c.length(5) == state[1][5] + 1


def test_batches_by_slot_are_scored_as_flat_ones(setting):
    """The pooling takes a batch as one (values, offsets) pair for each slot, too."""
    model, bb = setting
    a, b = _cache(model), _cache(model)
    flat = _batch(bb, [(0, 30)], [4, 20, 27])
    vo = flat["_val_offsets"].tolist() + [flat["_flat_values"].numel()]
    slots = {i + 1: (flat["_flat_values"][vo[i]:vo[i + 1]],
                     flat["_flat_row_offsets"].view(bb.features, -1)[i])
             for i in range(bb.features)}
    slots["user_offsets"] = flat["user_offsets"]
    want = model.predict_cached(flat, a, [2, 1])
    got = model.predict_cached(slots, b, [2, 1])
    assert torch.equal(got[4:27], want[4:27]) and got.shape == want.shape == (30,)
    assert _state(a) == _state(b)
