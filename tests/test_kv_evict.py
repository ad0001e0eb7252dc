"""Eviction by accumulated weight (gehtp_kv_evict): byte moves, equal to the rule stated position by position."""
import numpy as np
import pytest


def rule(w, n, keep, sinks, recent):
    """Positions of one key head that stay, in order."""
    if n <= keep:
        return list(range(n))
    value = lambda p: -np.inf if np.isnan(w[p]) else float(w[p])
    middle = sorted(range(sinks, n - recent), key=lambda p: (np.isnan(w[p]), -value(p), p))[:keep - sinks - recent]
    return list(range(sinks)) + sorted(middle) + list(range(n - recent, n))


class Call:
    def __init__(self, batch, kv_heads, d, slots, lengths, keep, sinks, recent, weights=None, seed=0):
        import torch
        r = np.random.default_rng(seed)
        self.shape = (batch, kv_heads, d, slots, keep, sinks, recent)
        self.ring = r.integers(-32768, 32767, (slots, 2, batch * kv_heads, d), np.int16, endpoint=True)
        self.w = r.standard_normal((batch, kv_heads, slots)).astype(np.float32) if weights is None else weights(r, (batch, kv_heads, slots)).astype(np.float32)
        self.n = np.array(lengths, np.int32)
        up = lambda a: torch.from_numpy(a.copy()).cuda()
        self.d_ring, self.d_w, self.d_n = up(self.ring), up(self.w), up(self.n)
        self.kept = torch.full((batch, kv_heads, keep), -7, dtype=torch.int32, device="cuda")

    def run(self, lib, in_place, kept=True):
        """in_place: caches, weights and lengths ("all"), or the lengths written elsewhere ("rows")."""
        import torch
        if in_place:
            self.o_ring, self.o_w, self.o_n = self.d_ring, self.d_w, self.d_n if in_place == "all" else torch.full_like(self.d_n, -1)
        else:
            self.o_ring, self.o_w, self.o_n = torch.full_like(self.d_ring, 77), torch.full_like(self.d_w, 9.0), torch.full_like(self.d_n, -1)
        ws = torch.full((lib.gehtp_kv_evict_workspace(*self.shape),), 255, dtype=torch.uint8, device="cuda")
        rc = lib.gehtp_kv_evict(self.d_ring.data_ptr(), self.o_ring.data_ptr(), self.d_w.data_ptr(), self.o_w.data_ptr(), self.d_n.data_ptr(), self.o_n.data_ptr(),
                                self.kept.data_ptr() if kept else None, *self.shape, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.gehtp_cuda_last_error()
        torch.cuda.synchronize()

    def check(self, in_place, kept=True):
        batch, kv_heads, d, slots, keep, sinks, recent = self.shape
        ring, w = (self.ring.copy(), self.w.copy()) if in_place else (np.full_like(self.ring, 77), np.full_like(self.w, 9.0))
        want = np.full((batch, kv_heads, keep), -1, np.int32)
        for b in range(batch):
            n = int(np.clip(self.n[b], 0, slots))
            for h in range(kv_heads):
                stay = rule(self.w[b, h], n, keep, sinks, recent)
                ring[:len(stay), :, b * kv_heads + h] = self.ring[stay, :, b * kv_heads + h]
                w[b, h, :len(stay)] = self.w[b, h, stay]
                if in_place:
                    w[b, h, len(stay):n] = 0.0
                want[b, h, :len(stay)] = stay
        assert np.array_equal(self.o_n.cpu().numpy(), np.minimum(np.clip(self.n, 0, slots), keep))
        if kept:
            assert np.array_equal(self.kept.cpu().numpy(), want)
        assert np.array_equal(self.o_w.cpu().numpy().view(np.int32), w.view(np.int32))
        assert np.array_equal(self.o_ring.cpu().numpy(), ring)


few = lambda r, s: r.integers(0, 3, s) * 0.5                                    # ties everywhere
odd = lambda r, s: r.choice([np.nan, -np.inf, np.inf, -0.0, 0.0, 1.0, -1.0, 1e-42, -1e-42], s)
CASES = [
    (1, 1, 8, 1, [1], 1, 0, 0, None), (1, 1, 64, 2, [2], 1, 0, 0, None), (2, 2, 64, 9, [0, 9], 4, 4, 0, None), (2, 2, 64, 9, [9, 5], 4, 0, 4, None),
    (3, 2, 80, 40, [40, 39, 3], 38, 1, 2, None), (2, 1, 128, 700, [700, 513], 512, 4, 64, few), (2, 3, 128, 1500, [1500, 1025], 1024, 0, 1000, odd),
    (5, 4, 128, 333, [333, -4, 400, 100, 101], 100, 7, 50, few), (1, 8, 128, 5000, [5000], 3000, 4, 256, None), (40, 2, 64, 130, [(3 * i) % 131 for i in range(40)], 64, 2, 8, odd),
    (1, 1, 512, 300, [299], 17, 0, 0, None), (2, 1, 128, 20000, [20000, 12345], 9000, 10, 100, few),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:4] + c[5:8])))
@pytest.mark.parametrize("in_place", [False, "rows", "all"])
def test_against_the_rule(cuda, case, in_place):
    call = Call(*case[:8], weights=case[8], seed=case[3])
    kept = case[0] != 3
    call.run(cuda, in_place, kept)
    call.check(in_place, kept)


@pytest.mark.gpu
def test_again_and_again(cuda):
    """A cache that is cut, grows and is cut again in place; a second call that finds nothing to do changes nothing."""
    import torch
    call = Call(3, 2, 64, 96, [96, 80, 40], 48, 2, 16, seed=3)
    for turn in range(4):
        call.run(cuda, "all")
        call.check("all")
        before = call.d_ring.clone(), call.d_w.clone(), call.d_n.clone()
        call.run(cuda, "all")
        assert torch.equal(before[0], call.d_ring) and torch.equal(before[1], call.d_w) and torch.equal(before[2], call.d_n)
        call.d_n += 30 - turn
        call.d_w += torch.rand_like(call.d_w)
        call.ring, call.w, call.n = (x.cpu().numpy() for x in (call.d_ring, call.d_w, call.d_n))


@pytest.mark.gpu
def test_captured_replayed_and_on_two_streams(cuda):
    import torch
    calls = [Call(5, 4, 128, 700, [700, 300, 650, 0, 699], 512, 4, 100, seed=1), Call(3, 2, 64, 90, [90, 89, 20], 40, 0, 8, weights=few, seed=2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graph = torch.cuda.CUDAGraph()

    def queue(call, stream):
        assert cuda.gehtp_kv_evict(call.d_ring.data_ptr(), call.o_ring.data_ptr(), call.d_w.data_ptr(), call.o_w.data_ptr(), call.d_n.data_ptr(), call.o_n.data_ptr(),
                                   call.kept.data_ptr(), *call.shape, call.ws.data_ptr(), call.ws.numel(), stream.cuda_stream) == 0
    for call in calls:
        call.ws = torch.empty(cuda.gehtp_kv_evict_workspace(*call.shape), dtype=torch.uint8, device="cuda")
        call.o_ring, call.o_w, call.o_n = torch.full_like(call.d_ring, 77), torch.full_like(call.d_w, 9.0), torch.full_like(call.d_n, -1)
    torch.cuda.synchronize()
    for _ in range(10):
        for call, stream in zip(calls, streams):
            queue(call, stream)
    torch.cuda.synchronize()
    for call in calls:
        call.check(False)
    a, b = calls[0], Call(5, 4, 128, 700, [1, 700, 513, 512, 600], 512, 4, 100, seed=9)
    with torch.cuda.graph(graph, stream=streams[0]):
        queue(a, streams[0])
    for x, y in ((a.d_ring, b.d_ring), (a.d_w, b.d_w), (a.d_n, b.d_n)):
        x.copy_(y)
    a.o_ring.fill_(77), a.o_w.fill_(9.0)
    graph.replay()
    torch.cuda.synchronize()
    a.ring, a.w, a.n = b.ring, b.w, b.n
    a.check(False)


@pytest.mark.gpu
def test_caches_past_four_gigabytes(cuda):
    """The last rows of a cache that is 4.3 GB long, in place and to another."""
    import torch
    batch, kvh, d, slots, keep = 64, 8, 128, 16500, 3
    ring = torch.zeros(slots, 2, batch * kvh, d, dtype=torch.int16, device="cuda")
    assert ring.numel() * 2 > 1 << 32
    ring[-2:] = torch.randint(-30000, 30000, ring[-2:].shape, dtype=torch.int16, device="cuda")
    want = ring[-2:].clone()
    w = torch.zeros(batch, kvh, slots, device="cuda")
    n = torch.full((batch,), slots, dtype=torch.int32, device="cuda")
    ws = torch.empty(cuda.gehtp_kv_evict_workspace(batch, kvh, d, slots, keep, 0, 2), dtype=torch.uint8, device="cuda")
    for out_n in (torch.zeros_like(n), n):
        out_ring = torch.zeros(slots, 2, batch * kvh, d, dtype=torch.int16, device="cuda") if out_n is not n else ring
        assert cuda.gehtp_kv_evict(ring.data_ptr(), out_ring.data_ptr(), w.data_ptr(), w.data_ptr(), n.data_ptr(), out_n.data_ptr(), None, batch, kvh, d, slots, keep, 0, 2,
                                   ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert (out_n == keep).all() and torch.equal(out_ring[1:3], want) and (out_ring[0] == 0).all()
        del out_ring


def test_workspace_refuses_what_the_call_refuses(cuda):
    ws = cuda.gehtp_kv_evict_workspace
    assert ws(2, 8, 128, 640, 512, 4, 64) >= 2 * 8 * 512 * 4
    for bad in ((0, 8, 128, 640, 512, 4, 64), (2, 0, 128, 640, 512, 4, 64), (65536, 1, 128, 640, 512, 4, 64), (2, 8, 4, 640, 512, 4, 64), (2, 8, 520, 640, 512, 4, 64),
                (2, 8, 128, 0, 0, 0, 0), (2, 8, 128, 640, 0, 0, 0), (2, 8, 128, 640, 641, 4, 64), (2, 8, 128, 640, 512, 449, 64), (2, 8, 128, 640, 512, 0xFFFFFFFF, 64)):
        assert ws(*bad) == 0 and b"kv evict" in cuda.gehtp_cuda_last_error()


@pytest.mark.parametrize("change,message", [
    (dict(ring=None), b"null"), (dict(out=None), b"null"), (dict(w=None), b"null"), (dict(wo=None), b"null"), (dict(n=None), b"null"), (dict(no=None), b"null"),
    (dict(ws=None), b"null"), (dict(ring=8), b"16-byte"), (dict(w=2), b"4-byte"), (dict(kept=2), b"4-byte"), (dict(ws=16), b"256-byte"), (dict(out=256), b"overlap"),
    (dict(wo=4), b"overlap"), (dict(no=4), b"overlap"), (dict(size=100), b"workspace"), (dict(), b"no memory of the current device"),
])
def test_refusals(cuda, change, message):
    buf = np.zeros(1 << 16, np.uint8)
    base = (buf.ctypes.data + 255) // 256 * 256
    at = lambda k: None if k in change and change[k] is None else base + change.get(k, 0)
    rc = cuda.gehtp_kv_evict(at("ring"), at("out"), at("w"), at("wo"), at("n"), at("no"), at("kept"), 2, 8, 128, 640, 512, 4, 64, at("ws"), change.get("size", 1 << 30), None)
    assert rc == -1 and message in cuda.gehtp_cuda_last_error()


@pytest.mark.gpu
def test_operands_that_overlap_are_refused(cuda):
    """Every pair of an output or the workspace with another operand but the one that it may be; nothing is queued."""
    import torch
    shape = (2, 4, 64, 40, 20, 1, 4)                           # batch, kv_heads, head_dim, slots, keep, sinks, recent
    ws = cuda.gehtp_kv_evict_workspace(*shape)
    size = dict(ring=40 * 8 * 64 * 4, ring_out=40 * 8 * 64 * 4, w=8 * 40 * 4, w_out=8 * 40 * 4, n=8, n_out=8, kept=8 * 20 * 4, ws=ws)
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
        return cuda.gehtp_kv_evict(at["ring"], at["ring_out"], at["w"], at["w_out"], at["n"], at["n_out"], at["kept"], *shape, at["ws"], ws,
                                   torch.cuda.current_stream().cuda_stream)
    assert call() == 0 and call(ring_out=place["ring"], w_out=place["w"], n_out=place["n"]) == 0
    torch.cuda.synchronize()
    before = buf.clone()
    unit = dict(ring_out=16, ws=256)
    for a in ("ring_out", "w_out", "n_out", "kept", "ws"):
        for b in size:
            if a == b or a == b + "_out":
                continue
            u = unit.get(a, 4)
            for start in (place[b], place[b] + (size[b] - 1) // u * u):
                assert call(**{a: start}) == -1 and b"overlap" in cuda.gehtp_cuda_last_error(), (a, b, start)
    torch.cuda.synchronize()
    assert torch.equal(before, buf)
