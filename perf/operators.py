"""Operators for a batch of sequences that go on from one prompt, measured one by one:

    shared    attention of a batch's new tokens over a prefix that all sequences share and the tail of each one's own,
              and, where asked for, the attention weight that every position of a tail has collected
    evict     the tails cut down to the positions of greatest weight
    verify    drafted tokens held against the target's probabilities, and the token that follows the accepted ones

A case is a dict of plain values. `prepare` makes its inputs on the GPU from a seed, `run` is one pass - in plain torch
operations, or where `own` is true through the library -, `exact` states in 64 bits what the pass computes.
"""
import math

import torch

own = False

TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
# query heads, key heads: grouped by 2, 4, 7, 8 and 16, one of each, and one key head for all
HEADS = [(16, 8), (32, 8), (14, 2), (28, 4), (64, 8), (32, 2), (8, 8), (16, 1), (12, 4)]


def _shared(name, batch, q_len, heads, dim, prefix, slots, fill, dtype, weights=False, joined=False):
    """fill: the tails are between fill * slots and slots long. joined: queries lie in rows of [q | k | v]."""
    return dict(name=name, kind="shared", batch=batch, q_len=q_len, heads=heads[0], kv_heads=heads[1], dim=dim, prefix=prefix, slots=slots, fill=fill,
                dtype=dtype, weights=weights, joined=joined)


def _evict(name, batch, kv_heads, dim, slots, fill, keep, sinks, recent, dtype):
    return dict(name=name, kind="evict", batch=batch, kv_heads=kv_heads, dim=dim, slots=slots, fill=fill, keep=keep, sinks=sinks, recent=recent, dtype=dtype)


def _verify(name, batch, drafts, vocab, dtype, temperature, with_draft=True, ragged=False):
    return dict(name=name, kind="verify", batch=batch, drafts=drafts, vocab=vocab, dtype=dtype, temperature=temperature, with_draft=with_draft, ragged=ragged)


def listed():
    return [
        # two answers to one short prompt, one token each: latency
        _shared("shared-b2-512", 2, 1, (16, 8), 128, 512, 64, 0.1, "float16"),
        # a small serving batch behind a long common document
        _shared("shared-b8-8k", 8, 1, (32, 8), 128, 8192, 512, 0.25, "float16"),
        # a full batch of samples from one very long prompt
        _shared("shared-b64-32k", 64, 1, (32, 8), 128, 32768, 1024, 0.1, "bfloat16"),
        # drafts of four verified at odd lengths, groups of seven heads of 64, queries inside the joined projection
        _shared("shared-b16-drafts-odd", 16, 5, (14, 2), 64, 4097, 333, 0.0, "bfloat16", joined=True),
        # drafts of seven for a full batch: many rows to every key
        _shared("shared-b64-drafts-16k", 64, 8, (32, 8), 128, 16384, 512, 0.25, "float16"),
        # long answers to a short prompt, with the weights that eviction goes by
        _shared("shared-b32-weights", 32, 1, (32, 8), 128, 2000, 4096, 0.25, "bfloat16", weights=True),
        # two tails a little over their budget
        _evict("evict-b2-640", 2, 8, 128, 640, 0.9, 512, 4, 64, "float16"),
        # a full batch cut to half
        _evict("evict-b64-2k", 64, 8, 128, 2048, 0.25, 1024, 4, 256, "bfloat16"),
        # one greedy request, drafts of four
        _verify("verify-b1-greedy", 1, 4, 32768, "float32", 0.0, with_draft=False),
        # a small batch with a draft model's logits
        _verify("verify-b8-sampled", 8, 5, 151936, "float16", 0.8),
        # a full batch, drafts of different lengths
        _verify("verify-b64-ragged", 64, 7, 151936, "bfloat16", 1.0, ragged=True),
        # drafts copied out of the prompt (no probabilities of their own), odd vocabulary, fp32 logits
        _verify("verify-b16-lookup", 16, 3, 50257, "float32", 0.7, with_draft=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    kind = rng.choice(["shared", "shared", "evict", "verify"])
    most = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        if kind == "shared":
            heads = rng.choice(HEADS)
            q_len = rng.choice([1, 1, 1, 2, 3, 4, 5, 6, 8])
            prefix = _log(rng, 1, 32768) if rng.random() < 0.9 else 0
            case = _shared("", _log(rng, 1, 64), q_len, heads, rng.choice([64, 128, 128]), prefix, _log(rng, 16, 4096), rng.choice([0.0, 0.25, 0.9]),
                           rng.choice(["float16", "bfloat16"]), rng.random() < 0.3, rng.random() < 0.3)
        elif kind == "evict":
            slots = _log(rng, 16, 8192)
            keep = max(1, int(slots * rng.uniform(0.2, 0.95)))
            sinks = min(rng.choice([0, 1, 4]), keep)
            case = _evict("", _log(rng, 1, 64), rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128]), slots, rng.choice([0.0, 0.25, 0.9]), keep, sinks,
                          int((keep - sinks) * rng.uniform(0.0, 0.6)), rng.choice(["float16", "bfloat16"]))
        else:
            case = _verify("", _log(rng, 1, 64), rng.randint(1, 8), _log(rng, 1000, 160000), rng.choice(["float32", "float16", "bfloat16"]),
                           rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]), rng.random() < 0.6, rng.random() < 0.5)
        del case["name"]
        if _cost(case) <= most:
            return case


def _spread(lo, hi, n):
    """n whole numbers spread evenly from lo to hi."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _lengths(case):
    return _spread(int(case["fill"] * case["slots"]), case["slots"], case["batch"])


def _draft_counts(case):
    return _spread(0, case["drafts"], case["batch"]) if case["ragged"] else [case["drafts"]] * case["batch"]


# ---------------------------------------------------------------- inputs


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = {"shared": _prepare_shared, "evict": _prepare_evict, "verify": _prepare_verify}[case["kind"]](case, gen)
    state["case"] = case
    return state


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _keys_values(gen, positions, heads, dim, lean):
    """[positions][keys, values][heads][dim]: keys of different lengths, the first leaning the way that queries do."""
    kv = _normal(gen, positions, 2, heads, dim)
    kv[:, 0] *= torch.exp(0.5 * _normal(gen, positions, heads, 1))
    if positions:
        kv[0, 0] += 2.0 * lean
    return kv


def _shuffled(gen, values):
    at = torch.randperm(len(values), generator=gen, device="cuda")
    return torch.tensor(values, dtype=torch.int32, device="cuda")[at]


def _prepare_shared(case, gen):
    b, t, h, kvh, d = (case[k] for k in ("batch", "q_len", "heads", "kv_heads", "dim"))
    dtype = TYPES[case["dtype"]]
    lean = _normal(gen, kvh, d)
    width = (h + 2 * kvh) * d if case["joined"] else h * d
    rows = _normal(gen, b * t, width)
    rows[:, : h * d] += 0.5 * lean.repeat_interleave(h // kvh, 0).reshape(1, -1)
    state = dict(q=rows.to(dtype), q_stride=width, n_tail=_shuffled(gen, _lengths(case)), prefix=_keys_values(gen, case["prefix"], kvh, d, lean).to(dtype),
                 tail=_keys_values(gen, case["slots"], b * kvh, d, lean.repeat(b, 1)).to(dtype), out=torch.zeros(b, t, h, d, dtype=dtype, device="cuda"),
                 scale=1.0 / math.sqrt(d))
    if case["weights"]:
        state["weights_in"] = torch.rand(b, kvh, case["slots"], generator=gen, device="cuda").square_() * 4.0
        state["weights"] = torch.zeros_like(state["weights_in"])
    return state


def _prepare_evict(case, gen):
    b, kvh, d, slots = (case[k] for k in ("batch", "kv_heads", "dim", "slots"))
    # what attention leaves behind: a few positions with most of the weight, some that never had any
    weights = torch.exp(2.0 * _normal(gen, b, kvh, slots))
    weights *= torch.rand(b, kvh, slots, generator=gen, device="cuda") > 0.1
    ring = _normal(gen, slots, 2, b * kvh, d).to(TYPES[case["dtype"]])
    return dict(ring=ring, weights=weights, n=_shuffled(gen, _lengths(case)), ring_out=torch.zeros_like(ring), weights_out=torch.zeros_like(weights),
                n_out=torch.zeros(b, dtype=torch.int32, device="cuda"), kept=torch.zeros(b, kvh, case["keep"], dtype=torch.int32, device="cuda"))


def _prepare_verify(case, gen):
    b, n, vocab, dtype, heat = case["batch"], case["drafts"], case["vocab"], TYPES[case["dtype"]], case["temperature"]
    target = (2.5 * _normal(gen, b, n + 1, vocab)).to(dtype)
    draft = (target[:, :n].float() + 0.7 * _normal(gen, b, n, vocab)).to(dtype)
    chosen = draft.float() / (heat or 1.0)
    if heat:
        chosen -= torch.log(-torch.log(torch.rand(b, n, vocab, generator=gen, device="cuda").clamp_(1e-20, 1.0 - 1e-7)))
    state = dict(target=target, tokens=chosen.argmax(-1).to(torch.int32), uniforms=torch.rand(b, n + 1, generator=gen, device="cuda"),
                 counts=_shuffled(gen, _draft_counts(case)), accepted=torch.zeros(b, dtype=torch.int32, device="cuda"),
                 out=torch.zeros(b, n + 1, dtype=torch.int32, device="cuda"))
    state["draft"] = draft if case["with_draft"] and heat else None
    return state


# ---------------------------------------------------------------- one pass


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"shared": _own_shared, "evict": _own_evict, "verify": _own_verify}[kind](state)
    return {"shared": _plain_shared, "evict": _plain_evict, "verify": _plain_verify}[kind](state)


def _address(t):
    return t.data_ptr() if t is not None and t.numel() else None


def _workspace(state, lib, size):
    """Held with the state, as a program holds it with its caches."""
    if "workspace" not in state:
        state["workspace"] = torch.empty(size(lib), dtype=torch.uint8, device="cuda")
    return state["workspace"].data_ptr(), state["workspace"].numel()


def _called(lib, rc):
    if rc:
        raise RuntimeError(lib.gehtp_cuda_last_error().decode())


def _own_shared(s):
    import gehtp_b200
    from gehtp_b200 import wtop
    lib, c = gehtp_b200.lib(), s["case"]
    shape = [c[k] for k in ("batch", "q_len", "heads", "kv_heads", "dim")]
    dt = wtop.DT_F16 if c["dtype"] == "float16" else wtop.DT_BF16
    ws, size = _workspace(s, lib, lambda lib: lib.gehtp_attn_shared_workspace(*shape, c["prefix"], c["slots"], int(c["weights"])))
    _called(lib, lib.gehtp_attn_shared(_address(s["q"]), _address(s["prefix"]), _address(s["tail"]), _address(s["n_tail"]), _address(s.get("weights_in")),
                                       _address(s.get("weights")), _address(s["out"]), *shape, s["q_stride"], c["prefix"], c["slots"], dt, s["scale"], ws, size,
                                       torch.cuda.current_stream().cuda_stream))
    return {"out": s["out"], "weights": s.get("weights")}


def _own_evict(s):
    import gehtp_b200
    lib, c = gehtp_b200.lib(), s["case"]
    shape = [c[k] for k in ("batch", "kv_heads", "dim", "slots", "keep", "sinks", "recent")]
    ws, size = _workspace(s, lib, lambda lib: lib.gehtp_kv_evict_workspace(*shape))
    _called(lib, lib.gehtp_kv_evict(_address(s["ring"]), _address(s["ring_out"]), _address(s["weights"]), _address(s["weights_out"]), _address(s["n"]),
                                    _address(s["n_out"]), _address(s["kept"]), *shape, ws, size, torch.cuda.current_stream().cuda_stream))
    return {"ring": s["ring_out"], "weights": s["weights_out"], "n": s["n_out"], "kept": s["kept"]}


def _own_verify(s):
    import gehtp_b200
    from gehtp_b200 import wtop
    lib, c = gehtp_b200.lib(), s["case"]
    dt = {"float32": wtop.DT_F32, "float16": wtop.DT_F16, "bfloat16": wtop.DT_BF16}[c["dtype"]]
    ws, size = _workspace(s, lib, lambda lib: lib.gehtp_verify_drafts_workspace(c["batch"], c["drafts"], c["vocab"]))
    _called(lib, lib.gehtp_verify_drafts(_address(s["target"]), _address(s["draft"]), _address(s["tokens"]), _address(s["counts"]), _address(s["uniforms"]),
                                         _address(s["accepted"]), _address(s["out"]), c["batch"], c["drafts"], c["vocab"], c["vocab"], c["vocab"], dt,
                                         c["temperature"], ws, size, torch.cuda.current_stream().cuda_stream))
    return {"accepted": s["accepted"], "out": s["out"]}


def _plain_shared(s):
    c = s["case"]
    b, t, h, kvh, d, n = (c[k] for k in ("batch", "q_len", "heads", "kv_heads", "dim", "slots"))
    rep, prefix = h // kvh, c["prefix"]
    # rows of a key head: [kvh][b][t][rep]
    q = s["q"][:, : h * d].float().reshape(b, t, kvh, rep, d).permute(2, 0, 1, 3, 4) * s["scale"]
    pk, pv = s["prefix"].float().permute(1, 2, 0, 3).unbind(0)
    tk, tv = s["tail"].float().reshape(n, 2, b, kvh, d).permute(1, 3, 2, 0, 4).unbind(0)
    at = torch.arange(n, device="cuda")
    ends = s["n_tail"][:, None] - t + 1 + torch.arange(t, device="cuda")              # what row t sees of its tail
    sees = (at < ends[..., None])[None, :, :, None, :]                               # [1][b][t][1][n]
    own_scores = torch.matmul(q.reshape(kvh, b, t * rep, d), tk.transpose(-1, -2)).reshape(kvh, b, t, rep, n)
    own_scores = torch.where(sees, own_scores, -math.inf)
    all_scores = torch.matmul(q.reshape(kvh, b * t * rep, d), pk.transpose(-1, -2)).reshape(kvh, b, t, rep, prefix)
    top = own_scores.amax(-1, keepdim=True)
    if prefix:
        top = torch.maximum(top, all_scores.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    own_scores = torch.exp(own_scores - top)
    all_scores = torch.exp(all_scores - top)
    total = own_scores.sum(-1, keepdim=True) + all_scores.sum(-1, keepdim=True)
    tv = torch.where((at < s["n_tail"][:, None])[None, :, :, None], tv, 0.0)
    out = torch.matmul(own_scores.reshape(kvh, b, t * rep, n), tv).reshape(kvh, b, t, rep, d)
    out = out + torch.matmul(all_scores.reshape(kvh, b * t * rep, prefix), pv).reshape(kvh, b, t, rep, d)
    total = torch.where(total == 0.0, 1.0, total)                                    # a row that sees nothing: zeros
    out = (out / total).permute(1, 2, 0, 3, 4).reshape(b, t, h, d)
    weights = None
    if c["weights"]:
        weights = s["weights_in"] + (own_scores / total).sum((2, 3)).permute(1, 0, 2)
        weights = torch.where((at < s["n_tail"][:, None])[:, None], weights, s["weights"])
    return {"out": out.to(s["out"].dtype), "weights": weights}


def _plain_evict(s):
    c = s["case"]
    b, kvh, d, slots, keep = (c[k] for k in ("batch", "kv_heads", "dim", "slots", "keep"))
    n = s["n"].long()[:, None, None]
    at = torch.arange(slots, device="cuda").expand(b, kvh, slots)
    always = (at < c["sinks"]) | (at >= n - c["recent"]) | (n <= keep)
    rank = torch.where(always, math.inf, s["weights"].double())
    rank = torch.where(at < n, rank, -math.inf)
    chosen = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    there = torch.arange(keep, device="cuda")
    chosen = torch.where(there < n, chosen, slots).sort(-1).values                    # in their order; places of no position last
    stays = chosen < slots                                                           # [b][kvh][keep]
    take = torch.where(stays, chosen, 0)
    kept = torch.where(stays, chosen, -1).to(torch.int32)
    weights = s["weights_out"].clone()
    weights[..., :keep] = torch.where(stays, s["weights"].gather(-1, take), weights[..., :keep])
    ring = s["ring_out"].clone()
    rows = s["ring"].reshape(slots, 2, b, kvh, d).gather(0, take.permute(2, 0, 1)[:, None, :, :, None].expand(keep, 2, b, kvh, d))
    left = ring[:keep].reshape(keep, 2, b, kvh, d)
    ring[:keep] = torch.where(stays.permute(2, 0, 1)[:, None, :, :, None], rows, left).reshape(keep, 2, b * kvh, d)
    return {"ring": ring, "weights": weights, "n": s["n"].clamp(max=keep), "kept": kept}


def _first_best(x):
    """The lowest place of the largest value."""
    best = x == x.amax(-1, keepdim=True)
    return torch.where(best, torch.arange(x.shape[-1], device=x.device), x.shape[-1]).amin(-1)


def _plain_verify(s):
    """In 64 bits throughout: a draw next to the border of two tokens goes to the one the numbers say."""
    c = s["case"]
    b, n, vocab, heat = c["batch"], c["drafts"], c["vocab"], c["temperature"]
    tokens, counts = s["tokens"].long(), s["counts"].long()
    u = s["uniforms"].double()
    if heat == 0.0:
        best = _first_best(s["target"])
        passes = best[:, :n] == tokens
    else:
        p = torch.softmax(s["target"].double() / heat, -1)
        px = p[:, :n].gather(-1, tokens[..., None])[..., 0]
        if s["draft"] is None:
            passes = u[:, :n] < px
        else:
            q = torch.softmax(s["draft"].double() / heat, -1)
            passes = u[:, :n] * q.gather(-1, tokens[..., None])[..., 0] < px
    place = torch.arange(n, device="cuda")
    passes &= place < counts[:, None]
    accepted = passes.long().cumprod(1).sum(1)
    row = torch.arange(b, device="cuda")
    if heat == 0.0:
        last = best[row, accepted]
    else:
        rest = p[row, accepted]
        rejected = (accepted < counts)[:, None]
        at = accepted.clamp(max=n - 1)
        if s["draft"] is None:
            away = torch.zeros_like(rest).scatter_(1, tokens[row, at][:, None], 1.0)
            less = rest * (1.0 - away)
        else:
            less = (rest - q[row, at]).clamp(min=0.0)
        less = torch.where(less.sum(-1, keepdim=True) > 0, less, rest)
        rest = torch.where(rejected, less, rest)
        upto = rest.cumsum(-1)
        last = torch.searchsorted(upto, u[:, n:] * upto[:, -1:], right=True)[:, 0].clamp(max=vocab - 1)
    places = torch.arange(n + 1, device="cuda")
    out = torch.where(places < accepted[:, None], torch.nn.functional.pad(tokens, (0, 1)), -1)
    out = torch.where(places == accepted[:, None], last[:, None], out)
    return {"accepted": accepted.to(torch.int32), "out": out.to(torch.int32)}


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["kind"] == "shared":
        kvh, d = case["kv_heads"], case["dim"]
        rows = case["batch"] * case["q_len"] * case["heads"]
        tails, t = _lengths(case), case["q_len"]
        seen = sum(max(0, n - i) for n in tails for i in range(t))
        size = 2 * 2 * rows * d + 4 * kvh * d * (case["prefix"] + sum(tails))
        if case["weights"]:
            size += 2 * 4 * kvh * sum(tails)
        return {"bytes": size, "flops": 4 * d * (rows * case["prefix"] + case["heads"] * seen)}
    if case["kind"] == "evict":
        heads, before = case["kv_heads"], _lengths(case)
        after = sum(min(n, case["keep"]) for n in before)
        # weights read, those that stay written with their places; rows that stay read and written
        return {"bytes": heads * (4 * sum(before) + 8 * after + 2 * 2 * 2 * case["dim"] * after), "flops": heads * sum(before)}
    size = 4 if case["dtype"] == "float32" else 2
    counts = _draft_counts(case)
    rows = sum(counts) + case["batch"]
    if case["with_draft"] and case["temperature"]:
        rows += sum(counts)
    return {"bytes": rows * case["vocab"] * size + 16 * case["batch"] * (case["drafts"] + 1), "flops": 4 * rows * case["vocab"]}


# ---------------------------------------------------------------- the definition, in 64 bits


def exact(case, seed):
    with torch.no_grad():
        return {"shared": _exact_shared, "evict": _exact_evict, "verify": _exact_verify}[case["kind"]](case, prepare(case, seed))


def _exact_shared(case, s):
    """One sequence and key head after another, over the keys its rows see."""
    b, t, h, kvh, d = (case[k] for k in ("batch", "q_len", "heads", "kv_heads", "dim"))
    rep = h // kvh
    out = torch.zeros(b, t, h, d, dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if case["weights"] else None
    lengths = s["n_tail"].tolist()
    for k in range(kvh):
        pk, pv = s["prefix"][:, 0, k].double(), s["prefix"][:, 1, k].double()
        for i in range(b):
            n = lengths[i]
            tail = s["tail"][:n, :, i * kvh + k].double()
            keys, values = torch.cat([pk, tail[:, 0]]), torch.cat([pv, tail[:, 1]])
            q = s["q"][i * t:(i + 1) * t, k * rep * d:(k + 1) * rep * d].double().reshape(t * rep, d)
            scores = (q @ keys.T) * s["scale"]
            total = len(pk) + n
            hidden = torch.arange(total, device="cuda")[None] >= (total - t + 1 + torch.arange(t, device="cuda"))[:, None]
            hidden &= torch.arange(total, device="cuda")[None] >= len(pk)
            scores.masked_fill_(hidden.repeat_interleave(rep, 0), -math.inf)
            probs = torch.nan_to_num(torch.softmax(scores, -1)) if total else scores
            out[i, :, k * rep:(k + 1) * rep] = (probs @ values).reshape(t, rep, d)
            if weights is not None:
                weights[i, k, :n] = s["weights_in"][i, k, :n].double() + probs[:, len(pk):].sum(0)
    return {"out": out, "weights": weights}


def _exact_evict(case, s):
    b, kvh, keep, sinks, recent = (case[k] for k in ("batch", "kv_heads", "keep", "sinks", "recent"))
    ring, weights = s["ring_out"].double(), s["weights_out"].double()
    kept = torch.full((b, kvh, keep), -1, dtype=torch.int64)
    lengths, source = s["n"].tolist(), s["weights"].cpu().tolist()
    for i in range(b):
        for k in range(kvh):
            n, w = lengths[i], source[i][k]
            stay = list(range(n))
            if n > keep:
                middle = sorted(range(sinks, n - recent), key=lambda p: (-w[p], p))[: keep - sinks - recent]
                stay = list(range(sinks)) + sorted(middle) + list(range(n - recent, n))
            at = torch.tensor(stay, dtype=torch.int64, device="cuda")
            ring[: len(stay), :, i * kvh + k] = s["ring"][at, :, i * kvh + k].double()
            weights[i, k, : len(stay)] = s["weights"][i, k, at].double()
            kept[i, k, : len(stay)] = at.cpu()
    return {"ring": ring, "weights": weights, "n": torch.tensor([min(n, keep) for n in lengths]), "kept": kept}


def _exact_verify(case, s):
    b, n, vocab, heat = case["batch"], case["drafts"], case["vocab"], case["temperature"]
    counts, tokens, uniforms = s["counts"].tolist(), s["tokens"].tolist(), s["uniforms"].tolist()

    def chances(rows, i, j):
        x = rows[i, j].double() / heat
        e = torch.exp(x - x.max())
        return e / e.sum()

    accepted, out = [], []
    for i in range(b):
        row, j, rest = [-1] * (n + 1), 0, None
        while j < counts[i]:
            x = tokens[i][j]
            if heat == 0.0:
                if int((s["target"][i, j] == s["target"][i, j].max()).nonzero()[0]) != x:
                    break
            else:
                p = chances(s["target"], i, j)
                q = chances(s["draft"], i, j) if s["draft"] is not None else torch.nn.functional.one_hot(torch.tensor(x, device="cuda"), vocab).double()
                if not uniforms[i][j] * float(q[x]) < float(p[x]):
                    rest = (p - q).clamp(min=0.0)
                    rest = rest if float(rest.sum()) > 0 else p
                    break
            row[j] = x
            j += 1
        if heat == 0.0:
            row[j] = int((s["target"][i, j] == s["target"][i, j].max()).nonzero()[0])
        else:
            rest = chances(s["target"], i, j) if rest is None else rest
            upto = rest.cumsum(0)
            row[j] = min(vocab - 1, int((upto <= uniforms[i][n] * float(upto[-1])).sum()))
        accepted.append(j)
        out.append(row)
    return {"accepted": torch.tensor(accepted), "out": torch.tensor(out)}
