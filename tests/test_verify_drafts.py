"""Verification of drafts (gehtp_verify_drafts) against the rule in 64 bits.

Its answers are whole numbers. Random numbers nearer to a border than the arithmetic is exact would have two right answers: the test
of acceptance is fp32 (2^-18 covers sums and exponentials of the sizes here), the draw is in 64 bits. `rule` says how near the nearest
border was, and inputs that come nearer are drawn again before anything runs."""
import numpy as np
import pytest

from gehtp_b200.wtop import DT_BF16, DT_F16, DT_F32

DT = {"float32": DT_F32, "bfloat16": DT_BF16, "float16": DT_F16}


def chances(x, heat):
    """None: no distribution."""
    if np.isnan(x).any() or x.max() in (np.inf, -np.inf):
        return None
    e = np.exp((x - x.max()) / heat)
    return e / e.sum()


def rule(target, draft, tokens, n, u, heat):
    """One sequence: (accepted, row of out, nearness of the nearest border of a test, of the draw)."""
    most, vocab = len(target) - 1, target.shape[1]
    out, near, j = np.full(most + 1, -1, np.int64), np.inf, 0
    ok = lambda x: not np.isnan(x).any() and np.isfinite(x.max())
    if heat == 0.0:
        while j < n and ok(target[j]) and tokens[j] == target[j].argmax():
            out[j] = tokens[j]
            j += 1
        out[j] = target[j].argmax() if ok(target[j]) else -1
        return j, out, near, near
    less = 0.0
    while j < n:
        p, x = chances(target[j], heat), tokens[j]
        if draft is None:
            q = np.zeros(vocab)
            q[x if 0 <= x < vocab else []] = 1.0
        else:
            q = chances(draft[j], heat)
        if p is None or q is None or not 0 <= x < vocab:
            less = 0.0 if q is None else q
            break
        near = min(near, abs(u[j] * q[x] - p[x]) / max(p[x], 1e-300))
        if not u[j] * q[x] < p[x]:
            less = q
            break
        out[j] = x
        j += 1
    p = chances(target[j], heat)
    if p is None:
        return j, out, near, np.inf
    r = np.maximum(p - less, 0.0)
    r = r if r.sum() > 0 else p
    c = r.cumsum()
    goal = u[-1] * c[-1]
    out[j] = min(int((c <= goal).sum()), int(np.nonzero(r)[0][-1]))
    return j, out, near, np.abs(c - goal).min() / c[-1]


def make(batch, n, vocab, dtype, heat, with_draft, seed, spread=2.5, noise=0.7, pad=(0, 0)):
    import torch
    g = torch.Generator().manual_seed(seed)
    dt = getattr(torch, dtype)
    target = (spread * torch.randn(batch, n + 1, vocab + pad[0], generator=g)).to(dt)
    draft = torch.full((batch, n, vocab + pad[1]), 50.0).to(dt)
    draft[:, :, :vocab] = (target[:, :n, :vocab].float() + noise * torch.randn(batch, n, vocab, generator=g)).to(dt)
    chosen = draft[:, :, :vocab].float() / (heat or 1.0)
    if heat:
        chosen = chosen - torch.log(-torch.log(torch.rand(batch, n, vocab, generator=g).clamp(1e-20, 1 - 1e-7)))
    tokens = chosen.argmax(-1).to(torch.int32)
    uniforms = torch.rand(batch, n + 1, generator=g)
    return target, draft if with_draft else None, tokens, uniforms


def verify(lib, target, draft, tokens, counts, uniforms, vocab, heat, stream=None, shift=0):
    import torch
    batch, n = tokens.shape
    name = str(target.dtype).split(".")[1]

    def up(t):                                                   # `shift` elements behind a 16-byte boundary
        if t is None:
            return None
        flat = torch.zeros(t.numel() + shift, dtype=t.dtype, device="cuda")
        flat[shift:] = t.reshape(-1).cuda()
        return flat[shift:]
    a = lambda t: t.data_ptr() if t is not None and t.numel() else None
    t, d = up(target), up(draft)
    tok, cnt, uni = tokens.cuda(), counts.cuda() if counts is not None else None, uniforms.cuda()
    accepted, out = torch.full((batch,), -9, dtype=torch.int32, device="cuda"), torch.full((batch, n + 1), -9, dtype=torch.int32, device="cuda")
    ws = torch.full((lib.gehtp_verify_drafts_workspace(batch, n, vocab),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    rc = lib.gehtp_verify_drafts(a(t), a(d), a(tok), a(cnt), a(uni), a(accepted), a(out), batch, n, vocab, target.shape[-1], draft.shape[-1] if draft is not None else 0,
                                 DT[name], heat, a(ws), ws.numel(), stream if stream is not None else torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.gehtp_cuda_last_error()
    torch.cuda.synchronize()
    return accepted.cpu().numpy(), out.cpu().numpy()


def by_rule(target, draft, tokens, counts, uniforms, vocab, heat):
    got = [rule(target[b, :, :vocab].double().numpy(), draft[b, :, :vocab].double().numpy() if draft is not None else None, tokens[b].numpy(),
                int(np.clip(counts[b], 0, tokens.shape[1])) if counts is not None else tokens.shape[1], uniforms[b].double().numpy(), heat) for b in range(len(target))]
    return np.array([x[0] for x in got]), np.array([x[1] for x in got]), min(x[2] for x in got), min(x[3] for x in got)


CASES = [
    # batch, drafts, vocab, dtype, temperature, draft logits, pads, shift
    (1, 1, 1, "float32", 1.0, True, (0, 0), 0), (2, 1, 2, "bfloat16", 1.0, True, (0, 0), 1), (3, 2, 7, "float16", 0.7, True, (1, 2), 3),
    (9, 4, 1000, "float32", 0.8, True, (0, 0), 0), (9, 4, 1001, "float32", 0.8, True, (0, 3), 1), (9, 3, 1003, "bfloat16", 1.0, True, (2, 0), 5),
    (20, 5, 4099, "float16", 1.3, True, (0, 0), 1), (33, 0, 777, "float32", 1.0, False, (0, 0), 0), (12, 6, 5000, "float32", 0.6, False, (0, 0), 2),
    (2, 8, 70001, "bfloat16", 1.0, True, (0, 0), 0), (2, 2, 151936, "float16", 0.8, True, (64, 0), 0), (5, 64, 300, "float32", 1.0, True, (0, 0), 0),
    (33, 5, 3001, "float32", 0.0, False, (0, 0), 3), (2, 20, 30000, "bfloat16", 0.0, False, (0, 0), 1), (700, 2, 90, "float16", 0.0, False, (0, 0), 1),
    (700, 2, 90, "float32", 0.9, True, (0, 0), 1),
    (9, 4, 1001, "float32", 0.0, False, (0, 0), 1), (3, 8, 40000, "bfloat16", 0.0, False, (0, 0), 0), (4, 3, 20011, "float16", 0.0, True, (5, 0), 0),
    # more pieces of rows than warps that take them
    (700, 2, 5000, "bfloat16", 1.0, True, (0, 8), 0), (120, 7, 30011, "bfloat16", 0.9, True, (0, 0), 1), (1100, 3, 4000, "float32", 0.0, False, (0, 0), 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:6])))
def test_against_the_rule(cuda, case):
    import torch
    batch, n, vocab, dtype, heat, with_draft, pad, shift = case
    for noise in (0.0, 0.3, 1.5):                     # drafts that all pass, most, few
        for seed in range(20):
            target, draft, tokens, uniforms = make(batch, n, vocab, dtype, heat, with_draft, 100 * seed + vocab, noise=noise, pad=pad)
            counts = torch.tensor([(5 * b + seed) % (n + 3) - 1 for b in range(batch)], dtype=torch.int32) if vocab % 2 else None
            accepted, out, near, draw = by_rule(target, draft, tokens, counts, uniforms, vocab, heat)
            if near > 2.0 ** -18 and draw > 1e-11:
                break
        else:
            raise AssertionError("no inputs away from all borders")
        got = verify(cuda, target, draft, tokens, counts, uniforms, vocab, heat, shift=shift)
        assert np.array_equal(got[0], accepted) and np.array_equal(got[1], out)


@pytest.mark.gpu
def test_shares_of_many_draws(cuda):
    """4096 draws a call follow p whatever the draft says: the counts of accepted and drawn tokens together, 6 standard deviations."""
    import torch
    vocab, batch, heat = 12, 4096, 0.9
    g = torch.Generator().manual_seed(5)
    p_logits, q_logits = torch.randn(vocab, generator=g), torch.randn(vocab, generator=g)
    q = torch.softmax(q_logits.double() / heat, 0)
    total = np.zeros(vocab)
    for turn in range(4):
        tokens = torch.multinomial(q.float(), batch, replacement=True, generator=g).to(torch.int32)[:, None]
        target, draft = p_logits.expand(batch, 2, vocab).contiguous(), q_logits.expand(batch, 1, vocab).contiguous()
        accepted, out = verify(cuda, target, draft, tokens, None, torch.rand(batch, 2, generator=g), vocab, heat)
        total += np.bincount(out[:, 0], minlength=vocab)
    p = torch.softmax(p_logits.double() / heat, 0).numpy()
    m = total.sum()
    assert (np.abs(total - m * p) <= 6 * np.sqrt(m * p * (1 - p))).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heat", [0.0, 1.0])
def test_rows_without_a_distribution(cuda, heat):
    import torch
    target, draft, tokens, uniforms = make(8, 2, 500, "float32", heat, heat > 0, 11, noise=0.0)
    target[0, 0, 3] = float("nan")
    target[1, 1] = -float("inf")
    target[2, 2, 499] = float("nan")
    target[3, 0, 7] = float("inf")
    tokens[4, 0], tokens[5, 1] = -1, 500                        # ids outside the vocabulary
    target[6, :, 100:] = -float("inf")                            # tokens ruled out
    if heat:
        draft[7, 0, 0] = float("nan")
    accepted, out, near, draw = by_rule(target, draft, tokens, None, uniforms, 500, heat)
    assert heat == 0.0 or (near > 2.0 ** -18 and draw > 1e-11)
    got = verify(cuda, target, draft, tokens, None, uniforms, 500, heat)
    assert np.array_equal(got[0], accepted) and np.array_equal(got[1], out)
    assert out[0, 0] == -1 and out[1, 1] == -1 and out[2, 2] == -1 and out[3, 0] == -1 and accepted[4] == 0 and accepted[5] <= 1


@pytest.mark.gpu
def test_ends_of_the_draw(cuda):
    """0 draws the first possible token, 1 - 2^-24 and what should not come (1, above, no number) a possible one."""
    import torch
    target = torch.full((6, 1, 3000), -float("inf"))
    target[:, 0, 1000:2000] = torch.randn(1000, generator=torch.Generator().manual_seed(2))
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 7.0, float("nan"), -1.0])[:, None]
    accepted, out = verify(cuda, target, None, torch.zeros(6, 0, dtype=torch.int32), None, u, 3000, 1.0)
    assert (accepted == 0).all() and (out[:, 0] >= 1000).all() and (out[:, 0] < 2000).all() and out[0, 0] == 1000 and out[5, 0] == 1000 and out[2, 0] == 1999


def test_workspace_refuses_what_the_call_refuses(cuda):
    ws = cuda.gehtp_verify_drafts_workspace
    assert ws(4, 3, 1000) > 0 and ws(1, 0, 1) > 0
    for bad in ((0, 3, 1000), (4097, 3, 1000), (4, 65, 1000), (4, 3, 0), (4, 3, (1 << 30) + 1)):
        assert ws(*bad) == 0 and b"verify drafts" in cuda.gehtp_cuda_last_error()


@pytest.mark.parametrize("change,message", [
    (dict(target=None), b"null"), (dict(tokens=None), b"null"), (dict(uniforms=None), b"null"), (dict(accepted=None), b"null"), (dict(out=None), b"null"),
    (dict(ws=None), b"null"), (dict(target=2), b"boundaries of their type"), (dict(draft=2), b"boundaries of their type"), (dict(out=2), b"4-byte"),
    (dict(ws=64), b"256-byte"), (dict(ts=999), b"rows"), (dict(ds=999), b"rows"), (dict(dt=3), b"element type"), (dict(heat=-1.0), b"temperature"),
    (dict(heat=1e-9), b"temperature"), (dict(heat=float("nan")), b"temperature"), (dict(heat=float("inf")), b"temperature"), (dict(size=8), b"workspace"), (dict(accepted=-192), b"overlaps"), (dict(out=-516), b"overlaps"), (dict(out=-340), b"overlaps"),
    (dict(), b"no memory of the current device"),
])
def test_refusals(cuda, change, message):
    buf = np.zeros(1 << 16, np.uint8)
    base = (buf.ctypes.data + 255) // 256 * 256
    place = dict(target=0, draft=0, tokens=0, n=64, uniforms=128, accepted=256, out=512, ws=1024)
    at = lambda k: None if k in change and change[k] is None else base + change.get(k, 0) + place[k]
    rc = cuda.gehtp_verify_drafts(at("target"), at("draft"), at("tokens"), at("n"), at("uniforms"), at("accepted"), at("out"), 4, 3, 1000, change.get("ts", 1000),
                                  change.get("ds", 1000), change.get("dt", DT_F32), change.get("heat", 1.0), at("ws"), change.get("size", 1 << 30), None)
    assert rc == -1 and message in cuda.gehtp_cuda_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,noise", [("float32", 3e-5), ("float32", 1e-3), ("float16", 0.0), ("float32", 0.0)])
def test_rows_that_are_nearly_alike(cuda, dtype, noise):
    """A token outside the vocabulary is refused, and the draw is from the little that p is above q: where that is a hundredth of a percent, its
    sum's 2^-43 of p are 2^-29 of it. Equal rows: from p."""
    import torch
    for seed in range(20):
        target, draft, tokens, uniforms = make(12, 2, 3001, dtype, 0.9, True, 7 + seed, noise=noise)
        tokens[:, 0] = -1
        accepted, out, near, border = by_rule(target, draft, tokens, None, uniforms, 3001, 0.9)
        if border > 2.0 ** -26:
            break
    got = verify(cuda, target, draft, tokens, None, uniforms, 3001, 0.9)
    assert border > 2.0 ** -26 and np.array_equal(got[0], accepted) and np.array_equal(got[1], out)


@pytest.mark.gpu
@pytest.mark.parametrize("heat", [0.0, 0.8])
def test_captured_and_replayed(cuda, heat):
    """Logits, tokens, counts and random numbers are those of the replay."""
    import torch
    batch, n, vocab = 6, 4, 5003
    t, d, tok, u = (x.cuda() for x in make(batch, n, vocab, "bfloat16", heat, True, 1))
    cnt = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    accepted, out = torch.zeros(batch, dtype=torch.int32, device="cuda"), torch.zeros(batch, n + 1, dtype=torch.int32, device="cuda")
    ws = torch.full((cuda.gehtp_verify_drafts_workspace(batch, n, vocab),), 255, dtype=torch.uint8, device="cuda")
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        assert cuda.gehtp_verify_drafts(t.data_ptr(), d.data_ptr(), tok.data_ptr(), cnt.data_ptr(), u.data_ptr(), accepted.data_ptr(), out.data_ptr(), batch, n, vocab, vocab,
                                        vocab, DT_BF16, heat, ws.data_ptr(), ws.numel(), stream.cuda_stream) == 0
    for seed in range(2, 40):
        t2, d2, tok2, u2 = make(batch, n, vocab, "bfloat16", heat, True, seed, noise=0.4)
        cnt2 = torch.tensor([(seed + b) % (n + 1) for b in range(batch)], dtype=torch.int32)
        want, rows, near, border = by_rule(t2, d2, tok2, cnt2, u2, vocab, heat)
        if near <= 2.0 ** -18 or border <= 1e-11:
            continue
        for x, y in ((t, t2), (d, d2), (tok, tok2), (cnt, cnt2), (u, u2)):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(accepted.cpu().numpy(), want) and np.array_equal(out.cpu().numpy(), rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [300, 5003, 70001])
@pytest.mark.parametrize("u", [0.0, 1.0])
def test_ends_of_a_draw_from_a_few_tokens(cuda, dtype, vocab, u):
    """Rows that differ in two tokens only: what is left of all others is the rounding of two sums in 64 bits. The ends of the draw yield a token of the vocabulary,
    with next to nothing of max(p - q, 0) in front of it (behind it)."""
    import torch
    for seed in range(6):
        g = torch.Generator().manual_seed(seed)
        target = 2.5 * torch.randn(16, 2, vocab, generator=g)
        target[:, :, vocab // 2], target[:, :, vocab // 2 + 1] = 5.0, 3.0
        target = target.to(getattr(torch, dtype))
        draft = target[:, :1].clone()
        draft[:, :, vocab // 2], draft[:, :, vocab // 2 + 1] = 3.0, 5.0
        tokens = torch.full((16, 1), -1, dtype=torch.int32)
        accepted, out = verify(cuda, target, draft, tokens, None, torch.full((16, 2), u), vocab, 0.9)
        assert (accepted == 0).all() and (out[:, 0] >= 0).all() and (out[:, 0] < vocab).all()
        for b in range(16):
            r = np.maximum(chances(target[b, 0].double().numpy(), 0.9) - chances(draft[b, 0].double().numpy(), 0.9), 0.0)
            assert (r[:out[b, 0]].sum() if u == 0.0 else r[out[b, 0] + 1:].sum()) <= 1e-12


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,fill,heat", [("float32", float(np.finfo(np.float32).min), 1.0), ("bfloat16", -3.3895313892515355e38, 0.7), ("float16", -65504.0, 1e-4),
                                             ("float32", 1e30, 0.8), ("float32", -1e17, 1.0), ("float32", 7e20, 1.0),
                                             ("float32", -5e21, 0.8), ("float32", 1e23, 1.0)])
@pytest.mark.parametrize("with_draft", [False, True])
def test_rows_masked_to_one_value(cuda, dtype, fill, heat, with_draft):
    """Every logit the same, the type's lowest number among them: each token is as likely as the next. The drafts' rows have only their first third."""
    import torch
    batch, vocab = 24, 3001
    target = torch.full((batch, 2, vocab), fill).to(getattr(torch, dtype))
    draft = target[:, :1].clone()
    draft[:, :, 1000:] = -float("inf")
    for seed in range(20):
        g = torch.Generator().manual_seed(seed)
        tokens = torch.randint(0, 1000, (batch, 1), generator=g, dtype=torch.int32)
        tokens[::3] = -1
        uniforms = torch.rand(batch, 2, generator=g)
        accepted, out, near, border = by_rule(target, draft if with_draft else None, tokens, None, uniforms, vocab, heat)
        if near > 2.0 ** -18 and border > 1e-11:
            break
    got = verify(cuda, target, draft if with_draft else None, tokens, None, uniforms, vocab, heat)
    assert border > 1e-11 and np.array_equal(got[0], accepted) and np.array_equal(got[1], out)


@pytest.mark.gpu
def test_far_logits_at_a_low_temperature(cuda):
    """Numbers an eighth apart, 1803 powers of two at this temperature: all but the largest weigh nothing."""
    import torch
    target = torch.full((4, 1, 3000), 1048586.0 - 0.125)
    at = torch.tensor([0, 700, 1503, 2999])
    target[torch.arange(4), 0, at] = 1048586.0
    accepted, out = verify(cuda, target, None, torch.zeros(4, 0, dtype=torch.int32), None, torch.tensor([[0.0], [0.3], [0.9], [0.5]]), 3000, 1e-4)
    assert out[:, 0].tolist() == at.tolist()


@pytest.mark.gpu
def test_operands_that_overlap_are_refused(cuda):
    """Every pair of an output or the workspace with another operand; nothing is queued. What a greedy call does not read may lie anywhere."""
    import torch
    batch, n, vocab = 3, 2, 1000
    ws = cuda.gehtp_verify_drafts_workspace(batch, n, vocab)
    size = dict(target=9 * 1000 * 4, tokens=24, n=12, u=36, accepted=12, out=36, ws=ws, draft=(5 * 1010 + 1000) * 4)
    place, end = {}, 0
    for name, bytes_ in size.items():
        place[name] = end
        end = (end + bytes_ + 255) // 256 * 256
    buf = torch.zeros(end + ws, dtype=torch.uint8, device="cuda")
    base = buf.data_ptr()
    assert base % 256 == 0

    def call(heat=1.0, **moved):
        at = {k: base + v for k, v in place.items()}
        at.update({k: base + v for k, v in moved.items()})
        return cuda.gehtp_verify_drafts(at["target"], at["draft"], at["tokens"], at["n"], at["u"], at["accepted"], at["out"], batch, n, vocab, 1000, 1010, DT_F32, heat,
                                        at["ws"], ws, torch.cuda.current_stream().cuda_stream)
    assert call() == 0 and call(0.0, ws=place["draft"]) == 0
    torch.cuda.synchronize()
    before = buf.clone()
    for a in ("accepted", "out", "ws"):
        for b in size:
            if a != b:
                u = 256 if a == "ws" else 4
                for start in (place[b], place[b] + (size[b] - 1) // u * u):
                    assert call(**{a: start}) == -1 and b"overlap" in cuda.gehtp_cuda_last_error(), (a, b, start)
    torch.cuda.synchronize()
    assert torch.equal(before, buf)
