"""The 4-bit key/value cache's operators, as they are measured: appending tokens to the cache and
reading them back, reading whole histories, and attention of new tokens over the cache.

A cache holds pages of 64 tokens.  Each 32 consecutive values of a token's key (or value) in one
head are stored as 32 codes n in 0..15 with a 16-bit scale s and a 16-bit base b of the tensors'
type T:

    s = T((max - min) / 15)      b = T(min - 16 s)      n = clamp(round((x - b) / s) - 16, 0, 15)

(round to nearest, ties to even; n = 0 where s = 0) and stand for (16 + n) s + b.  Sequence i
holds kv_lens[i] tokens, the last cu_seqlens[i+1] - cu_seqlens[i] of them new; its token at
position p is token p % 64 of page page_table[i, p // 64].  Attention of the new token at position
p over the keys j <= p of its sequence (causal), or over all kv_lens[i] of them:

    out = sum_j softmax_j(q . k_j / sqrt(head_dim)) v_j
"""
import numpy as np
import torch

own = False

PAGE = 64
GROUP = 32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _case(name, op, dtype, seqs, new, cached, heads, kv_heads, head_dim, causal=True, lens_seed=0):
    return {"name": name, "op": op, "dtype": dtype, "seqs": seqs, "new_lo": new[0],
            "new_hi": new[1], "cached_lo": cached[0], "cached_hi": cached[1], "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "causal": causal, "lens_seed": lens_seed}


def listed():
    return [
        # One event of each of a few users joins their histories; latency.
        _case("write-one-event", "write", "bf16", 24, (1, 1), (15, 255), 8, 8, 32),
        # A batch of whole histories (the packed 16..256-token sequences of the CTR model) is cached.
        _case("write-histories", "write", "bf16", 2048, (16, 256), (0, 0), 8, 8, 32),
        # Long chunks join longer histories, ragged on both ends.
        _case("write-long", "write", "fp16", 3, (9001, 15013), (101, 5003), 32, 8, 128),
        # Every history of a batch is read back.
        _case("read-histories", "read", "bf16", 1024, (0, 0), (16, 256), 8, 8, 32),
        # Two long contexts are read back.
        _case("read-long", "read", "fp16", 2, (0, 0), (30011, 40009), 16, 4, 64),
        # The newest event of one user attends to the user's history; latency.
        _case("attend-one-user", "attend", "bf16", 1, (1, 1), (199, 199), 8, 8, 32),
        # The newest event of every user of a batch.
        _case("attend-users", "attend", "bf16", 2048, (1, 1), (15, 255), 8, 8, 32),
        # One token over one long context, grouped heads.
        _case("attend-long-one", "attend", "bf16", 1, (1, 1), (131070, 131070), 32, 8, 128),
        # A batch of single tokens over ragged contexts, grouped heads.
        _case("attend-batch", "attend", "bf16", 48, (1, 1), (1000, 8000), 32, 8, 128),
        # A few candidates per user, each scored over the whole history.
        _case("attend-candidates", "attend", "fp16", 96, (7, 61), (300, 2000), 16, 4, 64, False),
        # A prompt's next chunk over what is cached and itself.
        _case("attend-chunk", "attend", "bf16", 4, (701, 2048), (2000, 8000), 16, 4, 128),
        # A serving step: the new events of every user are appended, then attend.
        _case("step-users", "step", "bf16", 1024, (1, 8), (15, 255), 8, 8, 32),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    op = rng.choice(["write", "read", "attend", "attend", "step"])
    dtype = rng.choice(["bf16", "fp16"])
    head_dim = rng.choice([32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    # Tokens over all sequences; a key's and a value's elements stay below 100 million.
    most = min(250000, 100000000 // (kv_heads * head_dim))
    total = log_int(200, most)
    seqs = log_int(1, min(2048, max(1, total // 16)))
    each = max(2, total // seqs)
    shape = rng.choice(["one", "few", "chunk"])
    new = {"one": 1, "few": rng.randint(2, 24), "chunk": log_int(2, 1024)}[shape]
    new = min(new, each)
    if op == "read":
        new = 0
    if op == "write" and shape == "chunk":
        new = each
    # The plain form holds a score for each query, head and key.
    if op in ("attend", "step") and seqs * new * heads * 2 * each > 500000000:
        new = max(1, 500000000 // (seqs * heads * 2 * each))
    lo, hi = each // 2, each + each // 3
    return {"op": op, "dtype": dtype, "seqs": seqs, "new_lo": min(new, max(1, new // 2)),
            "new_hi": new, "cached_lo": 0 if op == "write" and new == each else lo,
            "cached_hi": hi, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "causal": rng.random() < 0.75, "lens_seed": rng.randrange(1 << 30)}


def _lens(case):
    """(new, total) tokens of each sequence; they belong to the case, whatever the seed."""
    r = np.random.RandomState(case["lens_seed"])
    n = r.randint(case["new_lo"], case["new_hi"] + 1, case["seqs"])
    c = r.randint(case["cached_lo"], case["cached_hi"] + 1, case["seqs"])
    if case["op"] == "read":
        return c, c  # the whole sequence is read
    return n, n + c


def _inputs(case, seed):
    """Keys, values and queries of every token, on the GPU."""
    dt, h, d = DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"]
    new, total = _lens(case)
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    t = int(total.sum())
    # Keys have channels of their own size and offset, as learned projections give; values less so.
    k = normal(t, h, d).mul_(torch.exp(0.5 * normal(h, d))).add_(0.7 * normal(h, d)).to(dt)
    v = normal(t, h, d).mul_(torch.exp(0.2 * normal(h, d))).to(dt)
    q = normal(int(new.sum()), case["heads"], d).to(dt)
    pages = -(-total // PAGE)
    order = torch.randperm(int(pages.sum()), generator=g, device="cuda").to(torch.int32)
    first = np.cumsum(pages) - pages
    width = int(pages.max())
    at = torch.from_numpy(first[:, None] + np.minimum(np.arange(width), pages[:, None] - 1)).cuda()
    return k, v, q, order[at]


def _offsets(lens):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(lens)])).to(device="cuda",
                                                                       dtype=torch.int32)


def _new_rows(case):
    """Rows of the new tokens among all tokens, in order."""
    new, total = _lens(case)
    ends = np.cumsum(total)
    keep = np.ones(int(ends[-1]), dtype=bool)
    step = np.zeros(keep.size + 1, dtype=np.int64)
    np.add.at(step, ends - total, 1)
    np.add.at(step, ends - new, -1)
    keep = np.cumsum(step)[:-1] == 0
    return torch.from_numpy(np.nonzero(keep)[0]).cuda()


# ---------------------------------------------------------------------------
# The plain forms.
# ---------------------------------------------------------------------------
def _places(cu, kv_lens, table, tokens):
    """(page, slot) of each of the packed new tokens."""
    t = torch.arange(tokens, device=cu.device)
    s = torch.searchsorted(cu, t, right=True, out_int32=False) - 1
    p = (kv_lens[s] - (cu[s + 1] - cu[s])).long() + (t - cu[s])
    return table[s, p // PAGE].long(), p % PAGE


def _quantise(x):
    """Codes, scales and bases of x [tokens, heads, head_dim]; 64 bits, for the values next to a
    border between two codes."""
    y = x.double().unflatten(-1, (-1, GROUP))
    lo, hi = y.amin(-1), y.amax(-1)
    s = ((hi - lo) / 15).to(x.dtype)
    b = (lo - 16 * s.double()).to(x.dtype)
    sd, bd = s.double().unsqueeze(-1), b.double().unsqueeze(-1)
    n = (torch.round((y - bd) / torch.where(sd > 0, sd, 1.0)) - 16).clamp(0, 15)
    n = torch.where(sd > 0, n, 0.0).flatten(-2).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), s, b


def _values(codes, s, b):
    """What codes [..., head_dim / 2] stand for, in 32 bits."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    return ((16 + n) * s.float().unsqueeze(-1) + b.float().unsqueeze(-1)).flatten(-2)


def _plain_cache(case, num_pages):
    dt, h, d = DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"]
    codes = torch.zeros(2, num_pages, PAGE, h, d // 2, dtype=torch.uint8, device="cuda")
    return codes, torch.zeros(2, 2, num_pages, PAGE, h, d // GROUP, dtype=dt, device="cuda")


def _plain_append(cache, k, v, cu, kv_lens, table):
    codes, meta = cache
    page, slot = _places(cu, kv_lens, table, k.shape[0])
    nk, sk, bk = _quantise(k)
    nv, sv, bv = _quantise(v)
    codes[:, page, slot] = torch.stack([nk, nv])
    meta[:, :, page, slot] = torch.stack([torch.stack([sk, bk]), torch.stack([sv, bv])])


def _plain_read(cache, cu, kv_lens, table, tokens):
    codes, meta = cache
    page, slot = _places(cu, kv_lens, table, tokens)
    k = _values(codes[0, page, slot], meta[0, 0, page, slot], meta[0, 1, page, slot])
    v = _values(codes[1, page, slot], meta[1, 0, page, slot], meta[1, 1, page, slot])
    return k.to(meta.dtype), v.to(meta.dtype)


def _plain_attention(q, cache, cu, kv_lens, table, most_new, causal):
    """Every sequence padded to the longest; scores and softmax in 32 bits."""
    codes, meta = cache
    t, h, d = q.shape
    kvh = codes.shape[3]
    page = table.long()
    # [seqs, pages, 64, kv_heads, d] -> [seqs, kv_heads, keys, d]
    k = _values(codes[0][page], meta[0, 0][page], meta[0, 1][page]).flatten(1, 2).transpose(1, 2)
    v = _values(codes[1][page], meta[1, 0][page], meta[1, 1][page]).flatten(1, 2).transpose(1, 2)
    row = torch.arange(t, device=q.device)
    seq = torch.searchsorted(cu, row, right=True) - 1
    at = row - cu[seq]
    qp = torch.zeros(table.shape[0], most_new, h, d, device=q.device)
    qp[seq, at] = q.float()
    # [seqs, kv_heads, group, new, d]
    qp = qp.unflatten(2, (kvh, h // kvh)).permute(0, 2, 3, 1, 4)
    s = (qp.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (h // kvh, most_new)) / d ** 0.5
    key = torch.arange(k.shape[2], device=q.device)
    last = kv_lens.long()[:, None].expand(-1, most_new)
    if causal:
        first = kv_lens.long() - (cu[1:] - cu[:-1])
        last = torch.minimum(last, first[:, None] + torch.arange(most_new, device=q.device) + 1)
    seen = key < last[:, :, None]  # [seqs, new, keys]
    s = torch.where(seen[:, None, None], s, float("-inf"))
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e38))
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total, 0.0)
    o = (p.flatten(2, 3) @ v).unflatten(2, (h // kvh, most_new))
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, at].to(q.dtype)


# ---------------------------------------------------------------------------
# What is measured.
# ---------------------------------------------------------------------------
def prepare(case, seed):
    k, v, q, table = _inputs(case, seed)
    new, total = _lens(case)
    num_pages = int((-(-total // PAGE)).sum())
    st = {"case": case, "table": table, "cu": _offsets(new), "max_new": int(new.max()),
          "tokens": int(new.sum()), "max_kv": int(total.max()),
          "kv_lens": torch.from_numpy(total).to(device="cuda", dtype=torch.int32)}
    held = total - new if case["op"] in ("write", "step") else total  # cached before the pass
    if case["op"] in ("write", "step"):
        rows = _new_rows(case)
        st["k"], st["v"] = k[rows], v[rows]
        keep = torch.ones(k.shape[0], dtype=torch.bool, device="cuda")
        keep[rows] = False
        k, v = k[keep], v[keep]
    if case["op"] in ("attend", "step"):
        st["q"] = q
    held_lens = torch.from_numpy(held).to(device="cuda", dtype=torch.int32)
    if own:
        import cti_b200
        from cti_b200 import ops

        st["cache"] = cti_b200.KV4Cache(num_pages, case["kv_heads"], case["head_dim"],
                                        dtype=DTYPES[case["dtype"]], device="cuda")
        ops.kv4_append(st["cache"], k, v, _offsets(held), held_lens, table)
    else:
        st["cache"] = _plain_cache(case, num_pages)
        _plain_append(st["cache"], k, v, _offsets(held), held_lens, table)
    return st


def run(state):
    case, cache = state["case"], state["cache"]
    cu, lens, table = state["cu"], state["kv_lens"], state["table"]
    if own:
        from cti_b200 import ops

        if case["op"] in ("write", "step"):
            ops.kv4_append(cache, state["k"], state["v"], cu, lens, table)
        if case["op"] in ("write", "read"):
            return ops.kv4_read(cache, cu, lens, table, state["tokens"])
        return ops.kv4_attention(state["q"], cache, cu, lens, table, state["max_new"],
                                 causal=case["causal"], max_kv_len=state["max_kv"])
    if case["op"] in ("write", "step"):
        _plain_append(cache, state["k"], state["v"], cu, lens, table)
    if case["op"] in ("write", "read"):
        return _plain_read(cache, cu, lens, table, state["tokens"])
    return _plain_attention(state["q"], cache, cu, lens, table, state["max_new"], case["causal"])


def work(case):
    new, total = (x.astype(np.float64) for x in _lens(case))
    h, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    held = kvh * (d + 8 * (d // GROUP))  # bytes of a token's codes, scales and bases, K and V
    given = 2 * kvh * d * 2              # bytes of a token's keys and values in 16 bits
    t = float(new.sum())
    bytes_ = flops = 0.0
    if case["op"] == "write":
        bytes_ = t * (given + held + held + given)
        flops = t * kvh * d * 2 * 6.0
    elif case["op"] == "read":
        bytes_ = t * (held + given)
        flops = t * kvh * d * 2 * 2.0
    else:
        bytes_ = float(total.sum()) * held + t * h * d * 4
        pairs = new * total - (new * (new - 1) / 2 if case["causal"] else 0)
        flops = float(pairs.sum()) * h * d * 4
        if case["op"] == "step":
            bytes_ += t * (given + held)
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------
# The operators' definition in 64 bits, without pages.
# ---------------------------------------------------------------------------
def _stands_for(x):
    """The value that each element of x is held as."""
    t, h, d = x.shape
    y = x.to(torch.float64).reshape(t, h, d // GROUP, GROUP)
    low = y.min(dim=3, keepdim=True).values
    scale = ((y.max(dim=3, keepdim=True).values - low) / 15.0).to(x.dtype).to(torch.float64)
    base = (low - 16.0 * scale).to(x.dtype).to(torch.float64)
    steps = torch.where(scale > 0, (y - base) / scale, torch.full_like(y, 16.0))
    steps = torch.clamp(torch.round(steps), 16.0, 31.0)
    return (steps * scale + base).reshape(t, h, d)


def exact(case, seed):
    k, v, q, _ = _inputs(case, seed)
    if case["op"] in ("write", "read"):
        rows = _new_rows(case)
        return _stands_for(k[rows]), _stands_for(v[rows])
    new, total = _lens(case)
    group, d = case["heads"] // case["kv_heads"], case["head_dim"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    t0 = n0 = 0
    for n, length in zip(new.tolist(), total.tolist()):
        ks = _stands_for(k[t0:t0 + length]).repeat_interleave(group, dim=1)
        vs = _stands_for(v[t0:t0 + length]).repeat_interleave(group, dim=1)
        qs = q[n0:n0 + n].to(torch.float64)
        s = torch.einsum("nhd,lhd->hnl", qs, ks) * float(d) ** -0.5
        if case["causal"] and n > 1:
            i = torch.arange(length, device="cuda")
            s.masked_fill_(i[None, :] > (length - n) + i[:n, None], float("-inf"))
        out[n0:n0 + n] = torch.einsum("hnl,lhd->nhd", torch.softmax(s, dim=-1), vs)
        t0, n0 = t0 + length, n0 + n
    return out
