"""The CTR model's incremental forward on the 4-bit cache (SequenceCache, predict_cached): every
layer's attention against the plain 64-bit form on that layer's own queries and the histories of
its keys and values (bound: kv4_ref.attention), and the book-keeping around it."""
import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu


def _encoder(dev, layers=2, d=128, heads=4):
    from cti_b200.model import TransformerEncoder

    torch.manual_seed(3)
    enc = TransformerEncoder(d, heads, layers, 256, num_experts=8).to(dev).to(torch.bfloat16)
    for m in enc.moe:
        m.gate.float()
        m.prepare_for_inference()
    return enc


def _cache(enc, dev, seqs=4, pages=16, tokens=400):
    import cti_b200

    return cti_b200.SequenceCache(enc.num_layers, seqs, pages, enc.n_heads, enc.head_dim, tokens,
                                  device=dev)


def test_encoder_attends_to_what_each_layer_has_cached(cuda_device, monkeypatch):
    from cti_b200 import _lib, model

    dev = cuda_device
    enc = _encoder(dev)
    cache = _cache(enc, dev)
    history = [[[], [], [], []] for _ in range(enc.num_layers)]  # layer, sequence: (k, v) pieces
    step = {}
    plain = model.cached_attention
    calls = []

    def checked(q, k, v, layer_cache, extension):
        out = plain(q, k, v, layer_cache, extension)
        layer = cache.layers.index(layer_cache)
        calls.append(layer)
        at, ks, vs = 0, [], []
        for s, n in zip(step["seqs"], step["new"]):
            history[layer][s].append((k[at:at + n].cpu(), v[at:at + n].cpu()))
            ks += [p[0] for p in history[layer][s]]
            vs += [p[1] for p in history[layer][s]]
            at += n
        total = [cache.length(s) for s in step["seqs"]]
        want, tol = ref.attention(q.cpu(), ref.held(torch.cat(ks)), ref.held(torch.cat(vs)),
                                  step["new"], total, True, enc.head_dim ** -0.5)
        assert ((out.double().cpu() - want).abs() <= tol).all()
        return out

    monkeypatch.setattr(model, "cached_attention", checked)
    g = torch.Generator().manual_seed(0)
    for seqs, new in (([1, 3], [70, 1]), ([3, 0, 1], [1, 200, 0]), ([1], [1]), ([2, 1, 0, 3],
                                                                             [64, 3, 1, 130])):
        step.update(seqs=seqs, new=new)
        x = torch.randn(sum(new), enc.d_model, generator=g).bfloat16().to(dev)
        y, _ = enc(x, cache.extend(seqs, new))
        _lib.raise_on_status(dev)
        assert y.shape == x.shape and torch.isfinite(y).all()
    assert calls == [0, 1] * 4


def test_released_pages_serve_the_next_sequence(cuda_device):
    """A sequence on pages that another has used gives what it gives in a fresh cache."""
    dev = cuda_device
    enc = _encoder(dev)
    g = torch.Generator().manual_seed(1)
    a, b, c = (torch.randn(n, enc.d_model, generator=g).bfloat16().to(dev) for n in (150, 90, 5))
    fresh = _cache(enc, dev, pages=3)
    want = [enc(b, fresh.extend([0], [90]))[0], enc(c, fresh.extend([0], [5]))[0]]
    used = _cache(enc, dev, pages=3)
    enc(a, used.extend([2], [150]))
    used.release([2])
    got = [enc(b, used.extend([1], [90]))[0], enc(c, used.extend([1], [5]))[0]]
    for x, y in zip(want, got):
        assert torch.equal(x, y)


def test_encoder_refuses_a_cache_of_other_layers(cuda_device):
    enc = _encoder(cuda_device)
    cache = _cache(_encoder(cuda_device, layers=1), cuda_device)
    x = torch.zeros(2, enc.d_model, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(ValueError):
        enc(x, cache.extend([0], [2]))


def test_predict_cached_scores_the_new_tokens(cuda_device):
    """Histories in one call, then the new events in a second: the second returns the new events
    alone.  In 4 bits keys and values are off by up to half a step, 1/30 of their group's range; the
    configuration's weights (std 0.02) take that to far below 1e-2 in probability."""
    import cti_b200
    from cti_b200 import _lib, synth
    from cti_b200.model import build_ctr_model

    dev = cuda_device
    lens, new = [40, 100, 17], [1, 3, 2]
    total = sum(lens)
    bb = synth.bag_batch(batch=total, seed=4, vocab_hi=2e4)
    uo = torch.zeros(4, dtype=torch.int64)
    uo[1:] = torch.cumsum(torch.tensor(lens), 0)
    model = build_ctr_model(bb.vocab.tolist(), num_layers=2, num_experts=8, dim_ff=256)
    synth.init_ctr_model(model)
    with torch.no_grad():
        model.rep_encoder.emb.weight = torch.nn.Parameter(
            synth.embedding_table(bb.total_rows, 64, seed=1), requires_grad=False)
    model.to(dev).prepare_for_inference()
    batch = {"_flat_values": bb.values, "_flat_row_offsets": bb.row_offsets,
             "_val_offsets": bb.val_offsets, "user_offsets": uo}
    whole = model.predict(batch)

    def part(ranges):
        """The flat layout of some token ranges."""
        offs = bb.row_offsets.view(bb.features, total + 1)
        vals, ro, vo, start = [], [], [], 0
        for f in range(bb.features):
            base = int(bb.val_offsets[f])
            pieces = [bb.values[base + int(offs[f, a]):base + int(offs[f, b])] for a, b in ranges]
            counts = torch.cat([offs[f, a + 1:b + 1] - offs[f, a:b] for a, b in ranges])
            ro.append(torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(counts, 0)]))
            vals.append(torch.cat(pieces))
            vo.append(start)
            start += vals[-1].numel()
        n = torch.tensor([b - a for a, b in ranges])
        return {"_flat_values": torch.cat(vals), "_flat_row_offsets": torch.cat(ro),
                "_val_offsets": torch.tensor(vo),
                "user_offsets": torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(n, 0)])}

    starts = uo[:-1].tolist()
    ends = uo[1:].tolist()
    cache = model.sequence_cache(max_seqs=8, num_pages=10, max_tokens=256)
    first = model.predict_cached(part([(a, e - n) for a, e, n in zip(starts, ends, new)]), cache,
                                 [5, 0, 7])
    second = model.predict_cached(part([(e - n, e) for e, n in zip(ends, new)]), cache, [5, 0, 7])
    _lib.raise_on_status(dev)
    assert first.shape == (total - sum(new),) and second.shape == (sum(new),)
    rows = [e - n + j for e, n in zip(ends, new) for j in range(n)]
    assert (second - whole[rows]).abs().max() < 1e-2
    assert cti_b200.KV4Cache is type(cache.layers[0]) and cache.length(0) == 100
