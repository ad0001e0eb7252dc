"""Attention over a shared prefix and own tails (gehtp_attn_shared) against the formula in 64 bits.

Tolerance of an output component, from the roundings on the way to it, with A = sum p |v| of that component:
  eps/2 |out|                 the result's own rounding
  eps_p A                     the weights as matrix operands: fp16 2^-11; bf16 in two terms 2^-16
  2 e_s A                     the scores, once in the weight and once in the sum: head_dim fp32 additions of products whose magnitudes
                              sum up to S = scale * max_j sum |q k_j|, each off by 2^-23 of that at most, and the product with the scale
  2^-19 A                     the exponentials (2^-22) and the sums of weights and of partial results
  N 2^-24 max|v|              weights that fp16 holds with fewer bits (below 2^-14), N positions, against a sum of at least 1
"""
import ctypes

import numpy as np
import pytest

from gehtp_b200.wtop import DT_BF16, DT_F16, DT_F32

P = ctypes.c_void_p


def formula(q, prefix, tail, n_tail, scale):
    """q [b][t][h][d], prefix [P][2][kvh][d], tail [n][2][b * kvh][d] in 64 bits: out, its tolerance base A, S, weights of the tails."""
    import torch
    b, t, h, d = q.shape
    kvh = prefix.shape[2]
    rep = h // kvh
    out, mag = torch.zeros(b, t, h, d, dtype=torch.float64), torch.zeros(b, t, h, d, dtype=torch.float64)
    weights = torch.zeros(b, kvh, tail.shape[0], dtype=torch.float64)
    top = torch.zeros(b, t, h, 1, dtype=torch.float64)
    for i in range(b):
        for x in range(h):
            k = x // rep
            for y in range(t):
                n = max(0, int(n_tail[i]) - t + y + 1)
                keys = torch.cat([prefix[:, 0, k], tail[:n, 0, i * kvh + k]])
                values = torch.cat([prefix[:, 1, k], tail[:n, 1, i * kvh + k]])
                if not len(keys):
                    continue
                p = torch.softmax(keys @ q[i, y, x] * scale, 0)
                out[i, y, x], mag[i, y, x] = p @ values, p @ values.abs()
                top[i, y, x] = (keys.abs() @ q[i, y, x].abs()).max() * scale
                weights[i, k, :n] += p[len(prefix):]
    return out, mag, top, weights


def tolerance(out, mag, top, values, positions, dtype, d):
    import torch
    half, eps_p = (2.0 ** -11, 2.0 ** -11) if dtype == torch.float16 else (2.0 ** -8, 2.0 ** -16)
    tol = half * out.abs() + mag * (eps_p + 2 * top * (d + 2) * 2.0 ** -23 + 2.0 ** -19)
    return tol + (positions * 2.0 ** -24 * values.abs().max() + 2.0 ** -25 if dtype == torch.float16 else 1e-30)


class Call:
    """Operands of a call on the GPU; slots behind a tail's end hold NaN."""

    def __init__(self, batch, q_len, heads, kv_heads, d, prefix, slots, n_tail, dtype, weights=False, pad=0, seed=0):
        import torch
        g = torch.Generator().manual_seed(seed)
        self.shape, self.slots, self.n_prefix, self.dtype, self.scale = (batch, q_len, heads, kv_heads, d), slots, prefix, dtype, 1.0 / np.sqrt(d)
        r = lambda *s: torch.randn(*s, generator=g)
        self.stride = heads * d + pad
        rows = r(batch * q_len, self.stride)
        keys = torch.exp(0.7 * r(prefix + slots, 1, 1, 1))
        pre, tail = r(prefix, 2, kv_heads, d), r(slots, 2, batch * kv_heads, d)
        pre[:, 0] *= keys[:prefix, 0]
        tail[:, 0] *= keys[prefix:, 0]
        self.n = torch.tensor(n_tail, dtype=torch.int32)
        real = self.n.clamp(0, slots)
        for b in range(batch):
            tail.view(slots, 2, batch, kv_heads, d)[real[b]:, :, b] = float("nan")
        self.rows, self.prefix, self.tail = (x.to(dtype).cuda() for x in (rows, pre, tail))
        self.n_dev = self.n.cuda()
        self.out = torch.full((batch, q_len, heads, d), 7.0, dtype=dtype, device="cuda")
        self.w_in = torch.rand(batch, kv_heads, slots, generator=g).cuda() if weights else None
        self.w = torch.full_like(self.w_in, -5.0) if weights else None

    def size(self, lib):
        return lib.gehtp_attn_shared_workspace(*self.shape, self.n_prefix, self.slots, int(self.w is not None))

    def workspace(self, lib):
        import torch
        self.ws = torch.full((self.size(lib),), 255, dtype=torch.uint8, device="cuda")      # 255: every float in it NaN

    def run(self, lib, stream=None, w_in="own"):
        import torch
        a = lambda t: t.data_ptr() if t is not None and t.numel() else None
        if not hasattr(self, "ws"):
            self.workspace(lib)
        dt = DT_F16 if self.dtype == torch.float16 else DT_BF16
        rc = lib.gehtp_attn_shared(a(self.rows), a(self.prefix), a(self.tail), a(self.n_dev) if self.slots else None, a(self.w_in) if w_in == "own" else w_in,
                                   a(self.w), a(self.out), *self.shape, self.stride, self.n_prefix, self.slots, dt, self.scale, a(self.ws), self.ws.numel(),
                                   stream if stream is not None else torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.gehtp_cuda_last_error()

    def expected(self):
        """Of the operands as they are: result, weights, scores' sizes and the tolerance."""
        import torch
        b, t, h, kvh, d = self.shape
        q = self.rows.cpu().double()[:, :h * d].reshape(b, t, h, d)
        n = self.n.clamp(0, self.slots)
        tail = torch.nan_to_num(self.tail.cpu().double())
        want, mag, top, weights = formula(q, self.prefix.cpu().double(), tail, n, self.scale)
        values = torch.cat([self.prefix.cpu()[:, 1].reshape(-1), tail[:, 1].reshape(-1).to(self.dtype), torch.zeros(1, dtype=self.dtype)]).double()
        return want, weights, top, tolerance(want, mag, top, values, self.n_prefix + self.slots, self.dtype, d)

    def check(self):
        import torch
        torch.cuda.synchronize()
        b, t, h, kvh, d = self.shape
        n = self.n.clamp(0, self.slots)
        want, weights, top, tol = self.expected()
        got = self.out.cpu().double()
        assert torch.isfinite(got).all()
        off = (got - want).abs() - tol
        assert (off <= 0).all(), "%g over the tolerance at %s" % (off.max(), np.unravel_index(int(off.argmax()), off.shape))
        if self.w is not None:
            for i in range(b):
                assert (self.w[i, :, int(n[i]):] == -5.0).all()
                w, x = self.w[i, :, :int(n[i])].cpu().double(), self.w_in[i, :, :int(n[i])].cpu().double()
                rel = 2 * top[i].max() * (d + 2) * 2.0 ** -23 + 2.0 ** -19
                assert ((w - x - weights[i, :, :int(n[i])]).abs() <= weights[i, :, :int(n[i])] * rel + w.abs() * 2.0 ** -23 + 1e-30).all()


CASES = [
    # batch, q_len, heads, kv_heads, d, prefix, slots, n_tail
    (1, 1, 1, 1, 64, 1, 0, [0]),
    (1, 1, 4, 4, 128, 1, 1, [1]),
    (2, 1, 4, 2, 128, 0, 5, [0, 5]),                        # a sequence that sees nothing
    (3, 4, 14, 2, 64, 65, 70, [0, 3, 70]),                  # fewer positions than new tokens, groups of seven
    (3, 4, 14, 2, 64, 0, 70, [2, 3, 64]),                   # rows that see nothing
    (2, 1, 16, 1, 128, 63, 64, [64, 63]),
    (2, 16, 8, 1, 128, 130, 200, [16, 200]),                # 128 rows to a key head
    (1, 1, 71, 1, 64, 129, 129, [129]),
    (5, 2, 20, 4, 64, 1000, 333, [1, 64, 65, 128, 333]),
    (40, 1, 8, 1, 128, 300, 20, [i % 21 for i in range(40)]),
    (70, 5, 6, 2, 64, 127, 9, [i % 10 for i in range(70)]),
    (4, 1, 32, 8, 128, 2049, 3000, [3000, 1, 64, 1777]),
    (9, 8, 12, 4, 128, 513, 100, [-3, 1000, 8, 7, 9, 100, 64, 72, 71]),      # lengths outside the cache count as its ends
    (3, 2, 8, 2, 128, 0, 0, [0, 0, 0]),                     # nothing to see at all
    (20, 1, 16, 4, 128, 700, 0, [0] * 20),                  # no tails
    (33, 1, 16, 2, 128, 5000, 70, [i % 71 for i in range(33)]),              # two row tiles and a part of a third
    (12, 3, 28, 4, 64, 3000, 40, [(7 * i) % 41 for i in range(12)]),         # 18 tokens of seven heads to a row tile
    (4, 12, 10, 1, 128, 257, 150, [150, 13, 12, 11]),       # 120 rows to a tail
    (16, 1, 8, 1, 128, 513, 33, [33 - i for i in range(16)]),                # 128 rows that meet few positions: with the tails
    (1024, 1, 1, 1, 64, 5, 3, [i % 4 for i in range(1024)]),                 # the most sequences
    (130, 1, 2, 2, 64, 40, 300, [300 if i == 77 else 2 for i in range(130)]),
    (3, 4, 8, 4, 64, 70, 333, [333, 2, 47]),                # 8 rows to a tail
    (6, 1, 40, 8, 128, 0, 1500, [1500, 17, 0, 1, 16, 963]), # tails alone, slices that end inside 64 positions
    (50, 2, 9, 3, 128, 1000, 100, [(9 * i) % 101 for i in range(50)]),       # 6 rows to a tail beside the prefix's
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:7])))
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_against_the_formula(cuda, case, dtype):
    import torch
    call = Call(*case, dtype=getattr(torch, dtype), weights=case[6] > 0, pad=24, seed=len(case[7]) + case[5])
    call.run(cuda)
    call.check()


@pytest.mark.gpu
@pytest.mark.parametrize("prefix,rows", [(96, 1), (1500, 40)])
def test_again_and_without_given_weights(cuda, prefix, rows):
    """The same bits every time; weights_in NULL stands for zeros; in place adds up."""
    import torch
    call = Call(rows, 3, 8, 2, 128, prefix, 150, [(37 * i) % 151 for i in range(rows)], torch.bfloat16, weights=True)
    call.run(cuda, w_in=None)
    torch.cuda.synchronize()
    first = call.out.clone(), call.w.clone()
    for _ in range(5):
        call.ws.fill_(255)
        call.run(cuda, w_in=None)
        torch.cuda.synchronize()
        assert torch.equal(first[0].view(torch.int16), call.out.view(torch.int16)) and torch.equal(first[1], call.w)
    call.run(cuda, w_in=call.w.data_ptr())
    torch.cuda.synchronize()
    live = first[1] != -5.0
    assert torch.equal(call.w[live], 2 * first[1][live]) and (call.w[~live] == -5.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_a_position_that_is_no_number(cuda, dtype):
    """It makes no number of the rows that see it and of no others: not of earlier tokens, not of other sequences. Those may come by another
    order of sums, and are held to the formula."""
    import torch
    call = Call(3, 5, 8, 2, 128, 100, 90, [80, 70, 90], getattr(torch, dtype), weights=True)
    want, _, _, tol = call.expected()
    call.tail.view(90, 2, 3, 2, 128)[72, :, 0] = float("nan")        # the last but seven of the first sequence: seen by all its rows
    call.tail.view(90, 2, 3, 2, 128)[68, 1, 1, 0, 5] = float("inf")  # the second's last but one, a value: rows of the last two tokens
    call.tail.view(90, 2, 3, 2, 128)[88, 0, 2] = float("nan")        # the third's last but one, its key
    call.run(cuda)
    torch.cuda.synchronize()
    assert not torch.isfinite(call.out[0]).any()
    fine = (call.out.cpu().double() - want).abs() <= tol
    assert fine[1, :3].all() and fine[2, :3].all()
    assert not torch.isfinite(call.out[1, 3:, :4, 5]).any() and fine[1, 3:, 4:].all() and fine[1, 3:, :4, :5].all() and fine[1, 3:, :4, 6:].all()
    assert not torch.isfinite(call.out[2, 3:]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("prefix,d", [(3, 64), (700, 128)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_the_last_position_is_no_number(cuda, prefix, d, dtype):
    """As above with 8 rows to a tail: what only the last token sees."""
    import torch
    call = Call(20, 2, 8, 2, d, prefix, 90, [80, 70, 90] + [60] * 17, getattr(torch, dtype), weights=True)
    want, _, _, tol = call.expected()
    tail = call.tail.view(90, 2, 20, 2, d)
    tail[40, :, 0] = float("nan")
    tail[69, 1, 1, 0, 5] = float("inf")
    tail[89, 0, 2] = float("nan")
    call.run(cuda)
    torch.cuda.synchronize()
    assert not torch.isfinite(call.out[0]).any()
    fine = (call.out.cpu().double() - want).abs() <= tol
    assert fine[1, 0].all() and fine[2, 0].all() and fine[3:].all()
    assert not torch.isfinite(call.out[1, 1, :4, 5]).any() and fine[1, 1, 4:].all() and fine[1, 1, :4, :5].all() and fine[1, 1, :4, 6:].all()
    assert not torch.isfinite(call.out[2, 1]).any()


@pytest.mark.gpu
def test_captured_replayed_and_on_two_streams(cuda):
    """Lengths are read when the graph runs; calls on two streams with a workspace each."""
    import torch
    a = Call(6, 2, 8, 4, 128, 700, 200, [200, 1, 2, 64, 90, 3], torch.float16, weights=True)
    b = Call(33, 1, 16, 2, 64, 1200, 80, [(7 * i) % 81 for i in range(33)], torch.bfloat16, seed=4)
    a.run(cuda), b.run(cuda)
    torch.cuda.synchronize()
    want = a.out.clone(), a.w.clone(), b.out.clone()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for call, s in zip((a, b), streams):
            call.run(cuda, s.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(a.out, want[0]) and torch.equal(a.w, want[1]) and torch.equal(b.out, want[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        a.run(cuda, streams[0].cuda_stream)
    for seed in range(3):
        a.n = torch.tensor([(50 * seed + 31 * i) % 201 for i in range(6)], dtype=torch.int32)
        c = Call(6, 2, 8, 4, 128, 700, 200, a.n.tolist(), torch.float16, weights=True, seed=10 + seed)
        for x, y in ((a.rows, c.rows), (a.prefix, c.prefix), (a.tail, c.tail), (a.n_dev, c.n_dev), (a.w_in, c.w_in), (a.w, c.w)):
            x.copy_(y)
        graph.replay()
        a.check()


def test_workspace_refuses_what_the_call_refuses(cuda):
    ws = lambda *s: cuda.gehtp_attn_shared_workspace(*s)
    assert ws(2, 1, 16, 8, 128, 512, 64, 1) > ws(2, 1, 16, 8, 128, 512, 64, 0) > 0
    for bad in ((0, 1, 16, 8, 128, 512, 64, 0), (2, 0, 16, 8, 128, 512, 64, 0), (2, 1, 15, 8, 128, 512, 64, 0), (2, 1, 16, 0, 128, 512, 64, 0),
                (2, 1, 16, 8, 96, 512, 64, 0), (1025, 1, 16, 8, 128, 512, 64, 0), (2, 17, 16, 8, 128, 512, 64, 0), (2, 16, 9, 1, 128, 512, 64, 0),
                (2, 1, 16, 8, 128, 512, 0, 1), (2, 1, 16, 8, 128, (1 << 30) + 1, 64, 0), (2, 1, 16, 8, 128, 0, (1 << 24) + 1, 0), (1024, 1, 64, 64, 64, 1, 0, 0)):
        assert ws(*bad) == 0 and b"attn shared" in cuda.gehtp_cuda_last_error()


@pytest.mark.parametrize("change,message", [
    (dict(q=None), b"null"), (dict(out=None), b"null"), (dict(ws=None), b"null"), (dict(prefix=None), b"null"), (dict(tail=None), b"null"),
    (dict(n_tail=None), b"null"), (dict(w=None), b"weights_in"), (dict(w=64), b"overlap"), (dict(q=8), b"16-byte"), (dict(tail=8), b"16-byte"), (dict(ws=64), b"256-byte"),
    (dict(n_tail=2), b"4-byte"), (dict(stride=1024), b"q_stride"), (dict(stride=2052), b"q_stride"), (dict(dt=DT_F32), b"element type"),
    (dict(scale=0.0), b"scale"), (dict(scale=-1.0), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale"),
    (dict(size=1000), b"workspace"), (dict(heads=24, kv=16), b"shape"), (dict(), b"no memory of the current device"),
])
def test_refusals(cuda, change, message):
    """Host memory in every place: a call that got as far as its pointers says so, and nothing is queued."""
    buf = np.zeros(1 << 16, np.uint8)
    base = (buf.ctypes.data + 255) // 256 * 256
    at = lambda k: None if k in change and change[k] is None else base + change.get(k, 0)
    heads, kv = change.get("heads", 16), change.get("kv", 8)
    rc = cuda.gehtp_attn_shared(at("q"), at("prefix"), at("tail"), at("n_tail"), base, at("w"), at("out"), 2, 1, heads, kv, 128, change.get("stride", 2048), 512, 64,
                                change.get("dt", DT_F16), change.get("scale", 0.1), at("ws"), change.get("size", 1 << 40), None)
    assert rc == -1 and message in cuda.gehtp_cuda_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("batch,prefix", [(2, 700), (40, 3000), (140, 2000)])
@pytest.mark.parametrize("order", [1, -1])
def test_scores_that_outgrow_earlier_tiles(cuda, dtype, batch, prefix, order):
    """Keys that grow along the cache, or shrink: references raised behind a tile, within one, and never."""
    import torch
    call = Call(batch, 1, 8, 2, 128, prefix, 150, [(11 * i) % 151 for i in range(batch)], getattr(torch, dtype), weights=True, seed=batch)
    grow = torch.exp(order * torch.linspace(-2.25, 2.25, prefix + 150) + 0.25)
    call.prefix[:, 0] *= grow[:prefix, None, None].to(call.prefix)
    call.tail[:, 0] *= grow[prefix:, None, None].to(call.tail)
    call.run(cuda)
    call.check()


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 30, 60])
def test_prefix_position_that_is_no_number(cuda, batch):
    """All rows see the prefix: a key that is no number makes none of the rows of its head, an infinite value none of its component."""
    import torch
    call = Call(batch, 1, 8, 2, 128, 4000, 20, [i % 21 for i in range(batch)], torch.float16, seed=batch)
    want, _, _, tol = call.expected()
    call.prefix[1234, 0, 0] = float("nan")
    call.prefix[3999, 1, 1, 7] = float("inf")
    call.run(cuda)
    torch.cuda.synchronize()
    out = call.out.cpu().double()
    assert not torch.isfinite(out[:, :, :4]).any() and not torch.isfinite(out[:, :, 4:, 7]).any()
    rest = [i for i in range(128) if i != 7]
    assert ((out - want).abs() <= tol)[:, :, 4:, rest].all()


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [2, 24])
def test_caches_past_four_gigabytes(cuda, batch):
    """One key far behind the 2^32nd byte of the prefix, one of the tails, against zeros everywhere else."""
    import torch
    heads, kvh, d, prefix, slots = 16, 8, 128, (1 << 20) + 4097, (1 << 32) // (batch * 8 * 128 * 4) + 300
    q = torch.randn(batch, 1, heads, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    pre, tail = torch.zeros(prefix, 2, kvh, d, dtype=torch.bfloat16, device="cuda"), torch.zeros(slots, 2, batch * kvh, d, dtype=torch.bfloat16, device="cuda")
    n = torch.full((batch,), slots - 3, dtype=torch.int32, device="cuda")
    assert pre.numel() * 2 > 1 << 32 and tail.numel() * 2 > 1 << 32
    pre[prefix - 5, 0], pre[prefix - 5, 1] = 6.0, 3.0             # a key that queries meet by the sum of their components
    tail[slots - 4, 0], tail[slots - 4, 1] = -6.0, -5.0
    tail[slots - 3:] = float("nan")
    dots = q.cpu().double().sum(-1)[:, 0] * 6.0 * 0.125
    top = dots.abs()
    a, b, rest = torch.exp(dots - top), torch.exp(-dots - top), torch.exp(-top) * (prefix + slots - 3 - 2)
    want = (3.0 * a - 5.0 * b) / (a + b + rest)
    out = torch.zeros(batch, 1, heads, d, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(cuda.gehtp_attn_shared_workspace(batch, 1, heads, kvh, d, prefix, slots, 0), dtype=torch.uint8, device="cuda")
    rc = cuda.gehtp_attn_shared(q.data_ptr(), pre.data_ptr(), tail.data_ptr(), n.data_ptr(), None, None, out.data_ptr(), batch, 1, heads, kvh, d, heads * d, prefix, slots,
                                DT_BF16, 0.125, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, cuda.gehtp_cuda_last_error()
    torch.cuda.synchronize()
    got = out.cpu().double()[:, 0]
    # the scores as in `tolerance`, of one dot product; weights of the others are sums of a million equal terms, each sum 2^-24 a term off
    err = 2.0 ** -8 * want.abs() + (3 * a + 5 * b) / (a + b + rest) * (2.0 ** -16 + 2 * top * 130 * 2.0 ** -23 + 2.0 ** -19 + 2.0 ** -8)
    assert ((got - want[..., None]).abs() <= err[..., None] + 1e-30).all()
    assert cuda.gehtp_attn_shared_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("batch,q_len,heads,prefix", [(2, 3, 4, 0), (3, 4, 8, 60), (33, 2, 16, 700)])
def test_weights_beside_a_row_that_is_no_number(cuda, batch, q_len, heads, prefix):
    """The first token's query is no number, and so are the weights of the positions that it sees. Those behind them have theirs from the tokens that see them."""
    import torch
    call = Call(batch, q_len, heads, 2, 64, prefix, 90, [90 - i for i in range(batch)], torch.bfloat16, weights=True, seed=batch)
    _, weights, top, _ = call.expected()
    call.rows.view(batch, q_len, call.stride)[1, 0, :64] = float("nan")
    call.run(cuda)
    torch.cuda.synchronize()
    n = int(call.n[1])
    got = (call.w - call.w_in).cpu().double()
    assert torch.isnan(got[1, 0, :n - q_len + 1]).all()
    rel = 2 * top.max() * 66 * 2.0 ** -23 + 2.0 ** -19
    fine = lambda b, h, p: ((got[b, h, p] - weights[b, h, p]).abs() <= weights[b, h, p] * rel + call.w[b, h, p].cpu().abs() * 2.0 ** -22).all()
    assert fine(1, 0, slice(n - q_len + 1, n)) and fine(1, 1, slice(0, n)) and fine(0, 0, slice(0, int(call.n[0])))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("case", [
    (20, 1, 8, 8, 64, 9000, 0),             # a prefix on tcgen05, one row tile to a key head
    (36, 1, 8, 2, 128, 5000, 0),            # two
    (2, 1, 4, 2, 128, 0, 6000),             # tails of few rows
    (2, 4, 6, 1, 64, 0, 6000),              # of more
    (1, 1, 16, 1, 128, 3000, 3000),         # a prefix in the tails' launch
], ids=lambda c: "-".join(map(str, c)))
def test_many_small_weights_beside_a_large_one(cuda, case, dtype):
    """One position in 1024 has a score 26 bits above the others and the value 0: all of the result comes from weights of 2^-26. In fp16 a weight is off by at most
    2^-37 of the row's largest, or by its 11 bits: 2^-37 max|v| a position, over the sum of weights."""
    import torch
    batch, q_len, heads, kvh, d, prefix, slots = case
    call = Call(*case, [slots - 5 * i for i in range(batch)] if slots else [0] * batch, getattr(torch, dtype), seed=prefix)
    call.scale = 0.125
    call.rows.zero_()
    call.rows.view(batch * q_len, heads, d)[:, :, 0] = 8.0
    for cache, n in ((call.prefix, prefix), (call.tail, slots)):
        dead = torch.isnan(cache)
        cache[:, 0] = 0.0
        cache[::1024, 0, :, 0] = 18.0
        cache[:, 1] = 512.0 * (1.0 + (torch.arange(d, device="cuda") % 4) / 4).to(cache.dtype)
        cache[::1024, 1] = 0.0
        cache[dead] = float("nan")
    call.run(cuda)
    torch.cuda.synchronize()
    tail = torch.nan_to_num(call.tail.cpu().double())
    out, mag, top, _ = formula(call.rows.cpu().double().reshape(batch, q_len, heads, d), call.prefix.cpu().double(), tail, call.n, call.scale)
    half, eps_p, lost = (2.0 ** -11, 2.0 ** -11, 2.0 ** -37) if dtype == "float16" else (2.0 ** -8, 2.0 ** -16, 0.0)
    shortest = min(call.n.tolist()) - q_len + 1
    largest = (prefix + 1023) // 1024 + max(0, shortest + 1023) // 1024          # that every row sees
    tol = half * out.abs() + mag * (eps_p + 2 * top * (d + 2) * 2.0 ** -23 + 2.0 ** -19) + (prefix + slots) * lost * 896.0 / largest + 1e-30
    assert ((call.out.cpu().double() - out).abs() <= tol).all() and (out > 100 * (tol - half * out.abs() - mag * 2.0 ** -8)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("batch,prefix,slots", [(20, 3000, 0), (60, 3000, 70), (2, 0, 900), (3, 70, 70), (16, 100, 300)])
@pytest.mark.parametrize("order", ["any", "up", "down"])
@pytest.mark.parametrize("q", [4.0, 16384.0])
def test_scores_far_out(cuda, dtype, batch, prefix, slots, order, q):
    """Scores of up to 2^32, where neighbouring fp32 numbers are a factor of 2^512 apart as weights: the largest one is all of the row. Its weight's word of fp16 may be 2^-11
    off, beside a sum that is not (in bf16's two words 2^-16), and the result is rounded once more, where the weight is not 2^0 exactly."""
    import torch
    call = Call(batch, 2, 8, 2, 128, prefix, slots, [max(2, slots - i) for i in range(batch)] if slots else [0] * batch, getattr(torch, dtype), seed=batch)
    c = 3000.0 * torch.randn(prefix + slots, 2, generator=torch.Generator().manual_seed(prefix + slots))
    if order != "any":
        c = c.sort(0, descending=order == "down")[0]
    best = prefix // 2 if prefix else 1 if order == "down" else slots // 2     # a position that all rows of all sequences see
    c[best] = 25000.0
    call.rows.fill_(q)
    call.prefix[:, 0] = c[:prefix, :, None].to(call.prefix)
    dead = torch.isnan(call.tail)
    call.tail.view(slots, 2, batch, 2, 128)[:, 0] = c[prefix:, None, :, None].to(call.tail)
    call.tail[dead] = float("nan")
    call.run(cuda)
    torch.cuda.synchronize()
    value = call.prefix[best, 1][None] if prefix else call.tail[best, 1].view(batch, 2, 128)
    want = value.repeat_interleave(4, 1)[:, None].expand(batch, 2, 8, 128)
    eps = 2.0 ** -11 if dtype == "float16" else 2.0 ** -8
    eps += 2.0 ** -11 if dtype == "float16" else 2.0 ** -16
    got, want = call.out.double(), want.double()
    assert ((got - want).abs() <= want.abs() * (eps + 2.0 ** -19) + (2.0 ** -25 if dtype == "float16" else 0.0)).all()


@pytest.mark.gpu
def test_one_workspace_and_operands_replaced_before_every_call(cuda):
    """Calls of different sizes behind one another with the same workspace, each behind the copies that bring its operands."""
    import torch
    kinds = [(40, 3, 8, 2, 128, 1500, 150), (6, 1, 32, 8, 64, 4000, 0), (33, 1, 16, 2, 64, 1200, 80), (64, 8, 8, 1, 128, 300, 40), (3, 2, 8, 2, 128, 96, 90)]
    sets = []
    for i, kind in enumerate(kinds):
        calls = [Call(*kind, [(29 * x + 7 * turn) % (kind[6] + 1) for x in range(kind[0])], torch.float16, weights=kind[6] > 0, seed=10 * i + turn) for turn in range(3)]
        for c in calls:
            c.run(cuda)
        torch.cuda.synchronize()
        sets.append((Call(*kind, [0] * kind[0], torch.float16, weights=kind[6] > 0), calls))
    ws = torch.full((max(s[0].size(cuda) for s in sets),), 255, dtype=torch.uint8, device="cuda")
    got = []
    for turn in range(60):
        at, calls = sets[(turn * 3) % 5 if turn % 7 else turn % 5]
        c = calls[turn % 3]
        at.ws = ws
        for x, y in ((at.rows, c.rows), (at.prefix, c.prefix), (at.tail, c.tail), (at.n_dev, c.n_dev)):
            x.copy_(y)
        if c.w is not None:
            at.w_in.copy_(c.w_in), at.w.fill_(-5.0)
        at.run(cuda)
        got.append((c, at.out.clone(), at.w.clone() if c.w is not None else None))
    torch.cuda.synchronize()
    for c, out, w in got:
        assert torch.equal(out, c.out) and (w is None or torch.equal(w, c.w))


@pytest.mark.gpu
def test_operands_that_overlap_are_refused(cuda):
    """Every pair of an output or the workspace with another operand, by one byte at either end; nothing is queued."""
    import torch
    shape, prefix, slots = (2, 1, 16, 8, 128), 512, 64
    ws = cuda.gehtp_attn_shared_workspace(*shape, prefix, slots, 1)
    size = dict(q=4096 + 128 + 4096, prefix=prefix * 4096, tail=slots * 8192, n=8, w_in=4096, w=4096, out=8192, ws=ws)      # rows of q are 2112 elements apart
    place, end = {}, 0
    for name, bytes_ in size.items():
        place[name] = end
        end = (end + bytes_ + 255) // 256 * 256
    buf = torch.zeros(end + 512, dtype=torch.uint8, device="cuda")
    base = buf.data_ptr()
    assert base % 256 == 0

    def call(**moved):
        at = {k: base + v for k, v in place.items()}
        at.update({k: base + v for k, v in moved.items()})
        return cuda.gehtp_attn_shared(at["q"], at["prefix"], at["tail"], at["n"], at["w_in"], at["w"], at["out"], *shape, 2112, prefix, slots, DT_F16, 0.1, at["ws"], ws,
                                      torch.cuda.current_stream().cuda_stream)
    assert call() == 0, cuda.gehtp_cuda_last_error()
    assert call(w=place["w_in"]) == 0, cuda.gehtp_cuda_last_error()
    torch.cuda.synchronize()
    before = buf.clone()
    unit = dict(q=16, prefix=16, tail=16, out=16, ws=256)
    for a in ("out", "w", "ws"):
        for b in size:
            if a == b or {a, b} == {"w", "w_in"}:
                continue
            u = unit.get(a, 4)
            for start in (place[b], place[b] + (size[b] - 1) // u * u):
                assert call(**{a: start}) == -1 and b"overlap" in cuda.gehtp_cuda_last_error(), (a, b, start)
    torch.cuda.synchronize()
    assert torch.equal(before, buf)


@pytest.mark.parametrize("scale,message", [(3e38, b"scale"), (2.0 ** 127, b"no memory of the current device"), (1e-45, b"no memory of the current device")])
def test_scales_that_have_no_end_to_the_base_of_two(cuda, scale, message):
    """log2(e) times the scale has to be a number: a score of 0 would be none."""
    buf = np.zeros(1 << 16, np.uint8)
    at = (buf.ctypes.data + 255) // 256 * 256
    assert cuda.gehtp_attn_shared(at, at, at, at, None, None, at, 2, 1, 16, 8, 128, 2048, 512, 64, DT_F16, scale, at, 1 << 40, None) == -1 and message in cuda.gehtp_cuda_last_error()
