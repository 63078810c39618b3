"""The sequence operators' cases: attention of candidates (or of a sequence's own steps) over ragged behaviour histories with a learned
bucketed position bias, and the softmax cross entropy over a large item vocabulary.

`listed()` names the measured cases, `draw(rng)` makes others of the same ranges, `prepare(case, seed)` makes the device inputs and
`run(state)` is one pass: in plain torch operations (32 bits inside, rounded once at the end), or through the library's entry points when
the module's `own` is true.  `work(case)` counts what a pass cannot do without; `exact(case, seed)` is the definition in 64 bits."""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}


# ---- cases ---------------------------------------------------------------------------------------------------------------------------
def _attend(name, dtype, train, segments, max_q, max_k, heads, kv_heads, dim, causal=False, buckets=0, span=0, mask=False, own_keys=False,
            ragged=True, shape=0):
    return {"name": name, "op": "attend", "dtype": dtype, "train": train, "segments": segments, "max_q": max_q, "max_k": max_k, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "causal": causal, "buckets": buckets, "span": span, "mask": mask, "own_keys": own_keys,
            "ragged": ragged, "shape": shape}


def _vocab(name, dtype, train, rows, vocab, dim, bias=False, unlabelled=False):
    return {"name": name, "op": "vocab", "dtype": dtype, "train": train, "rows": rows, "vocab": vocab, "dim": dim, "bias": bias,
            "unlabelled": unlabelled}


def listed():
    return [
        # one impression: a single candidate attends to one user's short history -- what a latency-bound server runs per request
        _attend("one_candidate", "f32", False, 1, 1, 100, 2, 2, 16, mask=True, ragged=False),
        # one new event per user over long stored histories, heads sharing keys and values: the serving step of a sequence model
        _attend("next_event_long", "bf16", False, 48, 1, 16384, 8, 2, 64, causal=True, buckets=32, span=128),
        # ranking: a hundred or so candidates per user against that user's padded history
        _attend("rank_candidates", "f32", False, 32, 128, 500, 4, 4, 32, mask=True),
        # an odd head width, recency buckets, histories and candidate lists of odd sizes
        _attend("rank_odd_width", "bf16", False, 64, 129, 333, 4, 2, 40, buckets=20, span=100),
        # a training batch of the multi-hot models' shape (512 examples, up to 40 x 200 entries), f32 like the rest of the step
        _attend("train_short", "f32", True, 512, 40, 200, 4, 4, 16, buckets=16, span=64, mask=True),
        # next-event training over the whole history: every event attends to its predecessors
        _attend("train_history", "bf16", True, 8, 2048, 2048, 8, 8, 64, causal=True, buckets=32, span=128, own_keys=True),
        # a decoder's steps over an encoder's states of another length, wide heads that share keys
        _attend("train_encoder", "bf16", True, 16, 777, 1531, 8, 2, 128, mask=True),
        # a few users' scores against every feature of the 117,581-row vocabulary (the embedding width of the reference's DeepFM runs)
        _vocab("score_few", "f32", False, 4, 117581, 32),
        # held-out loss of a large batch
        _vocab("evaluate", "f32", False, 4096, 117581, 64, bias=True),
        # a training step's loss and gradients, f32
        _vocab("train_items", "f32", True, 1024, 117581, 64, bias=True, unlabelled=True),
        # the same over a million items in bf16: the logits alone would be 8 GB
        _vocab("train_million", "bf16", True, 2048, 1000000, 64),
        # odd sizes throughout, a wide embedding, log-popularity biases
        _vocab("train_odd", "bf16", True, 777, 50021, 200, bias=True, unlabelled=True),
    ]


def _between(rng, low, high):
    """A whole number, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.499)))))))


def draw(rng):
    dtype = rng.choice(["f32", "bf16"])
    train = rng.random() < 0.5
    most = max(work(c)["flops"] for c in listed())
    if rng.random() < 0.55:
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        dim = 8 * _between(rng, 1, 16)
        own_keys = rng.random() < 0.3
        max_q = 1 if rng.random() < 0.25 and not own_keys else _between(rng, 1, 2048)
        max_k = max_q if own_keys else _between(rng, 1, 2048 if max_q > 1 else 16384)
        buckets = rng.choice([0, 0, 2, 16, 32, 64])
        c = _attend("", dtype, train, _between(rng, 1, 512), max_q, max_k, heads, kv_heads, dim, causal=own_keys or rng.random() < 0.25,
                    buckets=buckets, span=_between(rng, max(1, buckets), 512) if buckets else 0, mask=rng.random() < 0.4, own_keys=own_keys,
                    ragged=rng.random() < 0.8, shape=rng.randrange(1 << 30))
        # a padded pass holds segments x heads x max_q x max_k scores: at most what the largest listed one does
        cells = max(x["segments"] * x["heads"] * x["max_q"] * x["max_k"] for x in listed() if x["op"] == "attend")
        while c["segments"] > 1 and (c["segments"] * heads * max_q * max_k > cells or work(c)["flops"] > most / 4):
            c["segments"] //= 2
    else:
        rows, vocab, dim = _between(rng, 1, 4096), _between(rng, 2, 1000000), 8 * _between(rng, 1, 32)
        c = _vocab("", dtype, train, rows, vocab, dim, bias=rng.random() < 0.5, unlabelled=rng.random() < 0.5)
        while c["rows"] > 1 and (c["rows"] * vocab > 5e8 or work(c)["flops"] > most / 4):
            c["rows"] //= 2
    del c["name"]
    return c


# ---- inputs --------------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """(queries, keys) of every segment: the case's alone, so that its work is."""
    rng = random.Random(case["shape"])
    pairs = []
    for i in range(case["segments"]):
        q, k = case["max_q"], case["max_k"]
        if case["ragged"] and i > 0:
            q = q if q == 1 else rng.randint(0, q)
            k = _between(rng, 1, k) if rng.random() < 0.95 else 0      # histories spread over orders of magnitude, some empty
        pairs.append((q, q if case["own_keys"] else k))
    return pairs


def _start(case, q, k):
    """Position of a segment's first query among its keys: its own step, or behind the history."""
    return 0 if case["own_keys"] else max(0, k - q)


def _boundaries(case):
    """Bucket borders of (key position - query position): single steps near zero, growing geometrically up to +-span."""
    n = case["buckets"] - 1
    if n < 1:
        return []
    if case["causal"]:
        sides = [-v for v in _grow(n, case["span"])]
    else:
        sides = [-v for v in _grow(n - n // 2, case["span"])] + [v + 1 for v in _grow(n // 2, case["span"])]
    return sorted(sides)


def _grow(n, span):
    steps = [min(i, n // 2) for i in range(n)]
    for i in range(n // 2 + 1, n):
        steps[i] = max(steps[i - 1] + 1, int(round((n // 2 + 1) * (max(span, n) / (n // 2 + 1)) ** ((i - n // 2) / max(1, n - 1 - n // 2)))))
    return [max(v, i) for i, v in enumerate(steps)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    t = TYPES[case["dtype"]]
    normal = lambda *size: torch.randn(size, generator=g, device=dev)   # noqa: E731
    s = {"case": case}
    if case["op"] == "attend":
        pairs = _lengths(case)
        random.Random(seed).shuffle(pairs)
        H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
        q_off, k_off = [0], [0]
        for q, k in pairs:
            q_off.append(q_off[-1] + q)
            k_off.append(k_off[-1] + k)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        s |= {"q_offsets": ints(q_off), "k_offsets": ints(k_off), "q_start": ints([_start(case, q, k) for q, k in pairs]),
              "total_q": q_off[-1], "total_k": k_off[-1]}
        s["q"] = normal(s["total_q"], H * D).to(t)
        s["k"] = normal(s["total_k"], Hk * D).to(t)
        s["v"] = normal(s["total_k"], Hk * D).to(t)
        s["keep"] = (torch.rand(s["total_k"], generator=g, device=dev) < 0.9).to(torch.uint8) if case["mask"] else None
        s["boundaries"] = _boundaries(case)
        s["bias"] = normal(case["buckets"], H) if case["buckets"] else None
        s["dout"] = normal(s["total_q"], H * D).to(t) if case["train"] else None
        s["scale"] = 1.0 / math.sqrt(D)
    else:
        N, V, D = case["rows"], case["vocab"], case["dim"]
        s["x"] = normal(N, D).to(t)
        s["w"] = (normal(V, D) * (2.0 / math.sqrt(D))).to(t)
        # popular items come first, as ids that were given by frequency rank do
        ranks = (torch.exp(torch.rand(N, generator=g, device=dev) * math.log(V)) - 1.0).long().clamp_(0, V - 1)
        if case["unlabelled"]:
            ranks = torch.where(torch.rand(N, generator=g, device=dev) < 0.1, -1, ranks)
        s["labels"] = ranks.to(torch.int32)
        s["bias"] = normal(V) * 0.5 - torch.log1p(torch.arange(V, device=dev)) * 0.3 if case["bias"] else None
        s["scale"] = 1.0 / N
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------------------
def run(state):
    if state["case"]["op"] == "attend":
        return _own_attend(state) if own else _plain_attend(state)
    return _own_vocab(state) if own else _plain_vocab(state)


def _rows(offsets, most, total):
    """Packed row of (segment, position), whether it is one, and the way back."""
    at = torch.arange(most, device=offsets.device)
    first, last = offsets[:-1, None].long(), offsets[1:, None].long()
    there = first + at < last
    row = torch.arange(total, device=offsets.device)
    seg = torch.searchsorted(offsets[1:].long(), row, right=True)
    return (first + at).clamp_(max=max(0, total - 1)), there, seg, row - offsets.long()[seg]


def _plain_attend(s):
    c = s["case"]
    B, H, Hk, D, mq, mk = c["segments"], c["heads"], c["kv_heads"], c["dim"], c["max_q"], c["max_k"]
    G = H // Hk
    t = s["q"].dtype
    iq, vq, sq, pq = _rows(s["q_offsets"], mq, s["total_q"])
    ik, vk, sk, pk = _rows(s["k_offsets"], mk, s["total_k"])
    if s["keep"] is not None:
        vk = vk & (s["keep"][ik] != 0)
    pad_q = lambda a: a.float()[iq].view(B, mq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * mq, D)          # noqa: E731
    pad_k = lambda a: torch.where(vk[..., None], a.float()[ik], 0.0).view(B, mk, Hk, D).permute(0, 2, 1, 3).contiguous()   # noqa: E731
    unpad_q = lambda a: a.view(B, H, mq, D).permute(0, 2, 1, 3).reshape(B, mq, H * D)[sq, pq].to(t)                   # noqa: E731
    unpad_k = lambda a: a.permute(0, 2, 1, 3).reshape(B, mk, Hk * D)[sk, pk].to(t)                                    # noqa: E731
    q, k, v = pad_q(s["q"]), pad_k(s["k"]), pad_k(s["v"])
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).view(B, H, mq, mk)
    rel = torch.arange(mk, device=q.device) - (s["q_start"][:, None].long() + torch.arange(mq, device=q.device))[..., None]
    borders = torch.tensor(s["boundaries"], device=q.device)
    if s["bias"] is not None:
        scores += s["bias"][torch.bucketize(rel, borders, right=True)].permute(0, 3, 1, 2)
    seen = vq[:, :, None] & vk[:, None, :]
    if c["causal"]:
        seen = seen & (rel <= 0)
    scores.masked_fill_(~seen[:, None], -math.inf)
    top = scores.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = scores.sub_(top).exp_()
    total = p.sum(3, keepdim=True)
    p /= torch.where(total == 0, 1.0, total)
    out = torch.matmul(p.view(B, Hk, G * mq, mk), v)
    result = {"out": unpad_q(out)}
    if not c["train"]:
        return result
    result["lse"] = (top + total.log()).squeeze(3).permute(0, 2, 1)[sq, pq]
    dout = pad_q(s["dout"])
    ds = torch.matmul(dout, v.transpose(2, 3)) - (dout * out).sum(3, keepdim=True)
    p = p.view(B, Hk, G * mq, mk)
    ds *= p
    result["dq"] = unpad_q(torch.matmul(ds, k) * s["scale"])
    result["dk"] = unpad_k(torch.where(vk[:, None, :, None], torch.matmul(ds.transpose(2, 3), q) * s["scale"], 0.0))
    result["dv"] = unpad_k(torch.where(vk[:, None, :, None], torch.matmul(p.transpose(2, 3), dout), 0.0))
    if s["bias"] is not None:
        # every diagonal's sum (a row's shift by one place brings equal distances under each other), then the buckets'
        skew = torch.nn.functional.pad(ds.view(B, H, mq, mk).flip(2), (0, mq)).flatten(2)[..., :mq * (mk + mq - 1)]
        along = skew.view(B, H, mq, mk + mq - 1).sum(2, dtype=torch.float64)
        far = torch.arange(mk + mq - 1, device=q.device) - (mq - 1) - s["q_start"][:, None].long()
        which = torch.bucketize(far, borders, right=True).flatten()
        hot = (which == torch.arange(c["buckets"], device=q.device)[:, None]).double()
        result["dbias"] = torch.matmul(hot, along.permute(0, 2, 1).reshape(-1, H)).float()
    return result


def _plain_vocab(s):
    c = s["case"]
    x, w = s["x"].float(), s["w"].float()
    labelled = s["labels"] >= 0
    label = s["labels"].long().clamp(min=0)[:, None]
    logits = torch.matmul(x, w.t())
    if s["bias"] is not None:
        logits += s["bias"]
    wanted = logits.gather(1, label)
    top = logits.amax(1, keepdim=True)
    p = logits.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    lse = top + total.log()
    result = {"loss": torch.where(labelled, (lse - wanted).squeeze(1), 0.0), "lse": lse.squeeze(1)}
    if not c["train"]:
        return result
    p /= total
    p.scatter_add_(1, label, torch.full_like(total, -1.0))
    p *= torch.where(labelled, s["scale"], 0.0)[:, None]
    result["dx"] = torch.matmul(p, w).to(s["x"].dtype)
    result["dw"] = torch.matmul(p.t(), x).to(s["w"].dtype)
    if s["bias"] is not None:
        result["dbias"] = p.sum(0)
    return result


def _own_attend(s):
    import ctypes as C
    from tf_repos_amd import capi
    c, lib = s["case"], capi.lib()
    H, Hk, D = c["heads"], c["kv_heads"], c["dim"]
    if "call" not in s:          # what a program keeps between calls: the description, the workspace and the outputs' buffers
        a = capi.Attention(dtype=capi.DTYPES[c["dtype"]], n_seg=c["segments"], heads=H, kv_heads=Hk, head_dim=D, max_q=c["max_q"],
                           max_k=c["max_k"], causal=int(c["causal"]), total_q=s["total_q"], total_k=s["total_k"], scale=s["scale"],
                           n_buckets=c["buckets"])
        a.boundaries[:len(s["boundaries"])] = s["boundaries"]
        size = C.c_int64()
        capi.check(lib.dctr_cross_attention_workspace_bytes(C.byref(a), int(c["train"]), C.byref(size)))
        dev = s["q"].device
        r = {"out": torch.empty_like(s["q"])}
        if c["train"]:
            r |= {"lse": torch.empty(s["total_q"], H, device=dev), "dq": torch.empty_like(s["q"]), "dk": torch.empty_like(s["k"]),
                  "dv": torch.empty_like(s["v"])}
            if s["bias"] is not None:
                r["dbias"] = torch.empty(c["buckets"], H, device=dev)
        s["call"] = (a, torch.empty(max(1, size.value), dtype=torch.uint8, device=dev), torch.zeros(2, dtype=torch.int32, device=dev), r)
    a, space, status, r = s["call"]
    p, st = capi.ptr, capi.current_stream()
    ins = (C.byref(a), p(s["q"]), H * D, p(s["k"]), Hk * D, p(s["v"]), Hk * D, p(s["q_offsets"]), p(s["k_offsets"]), p(s["q_start"]),
           p(s["keep"]), p(s["bias"]))
    capi.check(lib.dctr_cross_attention_fwd(*ins, p(r["out"]), H * D, p(r.get("lse")), p(status), p(space), space.numel(), st))
    if c["train"]:
        capi.check(lib.dctr_cross_attention_bwd(*ins, p(r["out"]), H * D, p(r["lse"]), p(s["dout"]), H * D, p(r["dq"]), H * D, p(r["dk"]), Hk * D,
                                                p(r["dv"]), Hk * D, p(r.get("dbias")), p(space), space.numel(), st))
    return r


def _own_vocab(s):
    import ctypes as C
    from tf_repos_amd import capi
    c, lib = s["case"], capi.lib()
    N, V, D, t = c["rows"], c["vocab"], c["dim"], capi.DTYPES[c["dtype"]]
    if "call" not in s:
        size = C.c_int64()
        capi.check(lib.dctr_vocab_softmax_workspace_bytes(t, N, V, D, int(c["train"]), C.byref(size)))
        dev = s["x"].device
        r = {"loss": torch.empty(N, device=dev), "lse": torch.empty(N, device=dev)}
        if c["train"]:
            r |= {"dx": torch.empty_like(s["x"]), "dw": torch.empty_like(s["w"])}
            if s["bias"] is not None:
                r["dbias"] = torch.empty(V, device=dev)
        s["call"] = (torch.empty(max(1, size.value), dtype=torch.uint8, device=dev), torch.zeros(2, dtype=torch.int32, device=dev), r)
    space, status, r = s["call"]
    p, st = capi.ptr, capi.current_stream()
    ins = (t, p(s["x"]), D, p(s["w"]), D, p(s["bias"]), p(s["labels"]), N, V, D, None, s["scale"])
    capi.check(lib.dctr_vocab_softmax_fwd(*ins, p(r["loss"]), p(r["lse"]), p(r.get("dx")), D, p(status), p(space), space.numel(), st))
    if c["train"]:
        capi.check(lib.dctr_vocab_softmax_bwd_weights(*ins, p(r["lse"]), p(r["dw"]), D, p(r.get("dbias")), p(space), space.numel(), st))
    return r


# ---- counts --------------------------------------------------------------------------------------------------------------------------
def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "attend":
        H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
        nq = nk = cells = 0
        for q, k in _lengths(case):
            nq, nk = nq + q, nk + k
            if case["causal"]:
                start = _start(case, q, k)
                whole = max(0, min(q, k - 1 - start)) if k else 0     # queries that do not see every key: start + i + 1 of them
                cells += whole * (start + 1) + whole * (whole - 1) // 2 + (q - whole) * k
            else:
                cells += q * k
        moved = size * D * (2 * nq * H + 2 * nk * Hk) + 4 * case["buckets"] * H + (nk if case["mask"] else 0)
        if case["train"]:
            moved += size * D * (2 * nq * H + 2 * nk * Hk) + 4 * nq * H + 4 * case["buckets"] * H
        return {"bytes": moved, "flops": cells * H * D * (14 if case["train"] else 4)}
    N, V, D = case["rows"], case["vocab"], case["dim"]
    once = size * D * (N + V) + (4 * V if case["bias"] else 0)
    return {"bytes": once * (2 if case["train"] else 1) + 12 * N, "flops": N * V * D * (6 if case["train"] else 2)}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attend(case, s) if case["op"] == "attend" else _exact_vocab(case, s)


def _exact_attend(c, s):
    H, Hk, D = c["heads"], c["kv_heads"], c["dim"]
    dev, f64 = s["q"].device, torch.float64
    qo, ko, start = s["q_offsets"].tolist(), s["k_offsets"].tolist(), s["q_start"].tolist()
    out = torch.zeros(s["total_q"], H, D, dtype=f64, device=dev)
    lse = torch.full((s["total_q"], H), -math.inf, dtype=f64, device=dev)
    dq, dk, dv = torch.zeros_like(out), torch.zeros(s["total_k"], Hk, D, dtype=f64, device=dev), torch.zeros(s["total_k"], Hk, D, dtype=f64, device=dev)
    dbias = torch.zeros(max(1, c["buckets"]), H, dtype=f64, device=dev)
    edges = torch.tensor([-(1 << 40)] + list(s["boundaries"]) + [1 << 40], device=dev)
    for b in range(c["segments"]):
        rows, cols = slice(qo[b], qo[b + 1]), slice(ko[b], ko[b + 1])
        n, m = qo[b + 1] - qo[b], ko[b + 1] - ko[b]
        if n == 0 or m == 0:
            continue
        q = s["q"][rows].to(f64).view(n, H, D).transpose(0, 1)
        k = s["k"][cols].to(f64).view(m, Hk, D).transpose(0, 1).repeat_interleave(H // Hk, 0)
        v = s["v"][cols].to(f64).view(m, Hk, D).transpose(0, 1).repeat_interleave(H // Hk, 0)
        z = s["scale"] * (q @ k.transpose(1, 2))
        where = start[b] + torch.arange(n, device=dev)
        spot = torch.arange(m, device=dev)
        # the keys of a query's bucket j are those from where + edges[j] up to where + edges[j + 1]: contiguous, so ranges are enough
        cut = (where[:, None] + edges).clamp(0, m)
        if c["buckets"]:
            size = cut[:, 1:] - cut[:, :-1]
            number = torch.repeat_interleave(torch.arange(c["buckets"], device=dev).repeat(n), size.flatten()).view(n, m)
            z = z + s["bias"].to(f64).t()[:, number]
        hide = torch.zeros(n, m, dtype=torch.bool, device=dev)
        if c["causal"]:
            hide |= spot > where[:, None]
        if s["keep"] is not None:
            hide |= s["keep"][cols] == 0
        z = z.masked_fill(hide, -math.inf)
        full = torch.logsumexp(z, 2)
        some = torch.isfinite(full)
        p = torch.exp(z - torch.where(some, full, 0.0)[..., None])
        o = p @ v
        out[rows], lse[rows] = o.transpose(0, 1), full.t()
        if c["train"]:
            go = s["dout"][rows].to(f64).view(n, H, D).transpose(0, 1)
            gp = go @ v.transpose(1, 2)
            gz = p * (gp - (p * gp).sum(2, keepdim=True))
            dq[rows] = (gz @ k).transpose(0, 1) * s["scale"]
            dk[cols] = (gz.transpose(1, 2) @ q).view(Hk, -1, m, D).sum(1).transpose(0, 1) * s["scale"]
            dv[cols] = (p.transpose(1, 2) @ go).view(Hk, -1, m, D).sum(1).transpose(0, 1)
            if c["buckets"]:
                run_up = torch.nn.functional.pad(gz.cumsum(2), (1, 0))
                ends = run_up.gather(2, cut.expand(H, n, -1))
                dbias += (ends[..., 1:] - ends[..., :-1]).sum(1).t()
    result = {"out": out.flatten(1)}
    if c["train"]:
        result |= {"lse": lse, "dq": dq.flatten(1), "dk": dk.flatten(1), "dv": dv.flatten(1)}
        if c["buckets"]:
            result["dbias"] = dbias
    return result


def _exact_vocab(c, s):
    f64 = torch.float64
    x, w = s["x"].to(f64), s["w"].to(f64)
    N = c["rows"]
    on = (s["labels"] >= 0).to(f64)
    at = s["labels"].long().clamp(min=0)
    loss, lse, dx, dw = torch.zeros(N, dtype=f64, device=x.device), torch.zeros(N, dtype=f64, device=x.device), torch.zeros_like(x), torch.zeros_like(w)
    db = torch.zeros(c["vocab"], dtype=f64, device=x.device)
    step = max(1, int(2.5e8) // c["vocab"])
    for i in range(0, N, step):
        rows = slice(i, min(N, i + step))
        z = x[rows] @ w.t()
        if c["bias"]:
            z += s["bias"].to(f64)
        lse[rows] = torch.logsumexp(z, 1)
        mine = torch.arange(z.shape[0], device=x.device), at[rows]
        loss[rows] = (lse[rows] - z[mine]) * on[rows]
        if c["train"]:
            z = torch.exp(z - lse[rows][:, None])
            z[mine] -= 1.0
            z *= (on[rows] * s["scale"])[:, None]
            dx[rows] = z @ w
            dw += z.t() @ x[rows]
            db += z.sum(0)
    result = {"loss": loss, "lse": lse}
    if c["train"]:
        result |= {"dx": dx, "dw": dw}
        if c["bias"]:
            result["dbias"] = db
    return result
