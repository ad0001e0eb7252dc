"""Answers to one prompt as a serving loop runs them: drafted tokens appended to every tail, attention over prefix and tails with the tails' weights,
drafts verified, tails rolled back to what was accepted, and cut when they are over their budget. Every operator's result is held to
its statement in 64 bits on the operands it had."""
import numpy as np
import pytest

import test_kv_evict
import test_shared_attn
import test_verify_drafts
from gehtp_b200.wtop import DT_BF16, DT_F16, DT_F32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,heat,batch,prefix", [("float16", 0.8, 5, 300), ("bfloat16", 0.0, 40, 700)])
def test_serving_loop(cuda, dtype, heat, batch, prefix):
    import torch
    heads, kvh, d, vocab, slots, keep, sinks, recent, drafts = 8, 2, 64, 211, 96, 40, 2, 16, 3
    g = torch.Generator().manual_seed(batch)
    dt = getattr(torch, dtype)
    r = lambda *s: torch.randn(*s, generator=g)
    eq, ek, ev = r(vocab, heads, d), r(vocab, kvh, d), r(vocab, kvh, d)
    head = r(heads * d, vocab).cuda() * 0.5
    pre = r(prefix, 2, kvh, d).to(dt).cuda()
    tail = torch.full((slots, 2, batch, kvh, d), float("nan"), dtype=dt, device="cuda")
    n, w = torch.zeros(batch, dtype=torch.int32, device="cuda"), torch.zeros(batch, kvh, slots, device="cuda")
    last = torch.randint(0, vocab, (batch,), generator=g)
    t = drafts + 1
    a = lambda x: x.data_ptr()
    scale, stream = 1.0 / np.sqrt(d), torch.cuda.current_stream().cuda_stream
    room = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for size in
            (cuda.gehtp_attn_shared_workspace(batch, t, heads, kvh, d, prefix, slots, 1), cuda.gehtp_verify_drafts_workspace(batch, drafts, vocab),
             cuda.gehtp_kv_evict_workspace(batch, kvh, d, slots, keep, sinks, recent))]
    kept = torch.zeros(batch, kvh, keep, dtype=torch.int32, device="cuda")
    cuts = passed = 0
    for step in range(48):
        # a draft that knows the target's last choices half of the time
        drafted = torch.randint(0, vocab, (batch, drafts), generator=g)
        tokens = torch.cat([last[:, None], drafted], 1)
        row = torch.arange(batch, device="cuda")
        for i in range(t):
            tail[n.long() + i, 0, row], tail[n.long() + i, 1, row] = ek[tokens[:, i]].to(dt).cuda(), ev[tokens[:, i]].to(dt).cuda()
        n += t
        q = eq[tokens].to(dt).cuda()
        out, before = torch.zeros(batch, t, heads, d, dtype=dt, device="cuda"), w.clone()
        assert cuda.gehtp_attn_shared(a(q), a(pre), a(tail), a(n), a(w), a(w), a(out), batch, t, heads, kvh, d, heads * d, prefix, slots,
                                      DT_F16 if dtype == "float16" else DT_BF16, scale, a(room[0]), room[0].numel(), stream) == 0, cuda.gehtp_cuda_last_error()
        target = (out.reshape(batch, t, -1).float() @ head).contiguous()
        draft = (target[:, :drafts] + 0.5 * torch.randn(batch, drafts, vocab, generator=g).cuda()).contiguous()
        if step % 2:                                              # what the draft model would have drawn: its own best
            drafted = draft.argmax(-1).cpu()
        tok, u = drafted.to(torch.int32).cuda(), torch.rand(batch, t, generator=g).cuda()
        accepted, chosen = torch.zeros(batch, dtype=torch.int32, device="cuda"), torch.zeros(batch, t, dtype=torch.int32, device="cuda")
        assert cuda.gehtp_verify_drafts(a(target), a(draft), a(tok), None, a(u), a(accepted), a(chosen), batch, drafts, vocab, vocab, vocab, DT_F32, heat, a(room[1]),
                                        room[1].numel(), stream) == 0, cuda.gehtp_cuda_last_error()
        torch.cuda.synchronize()
        # ---- against the statements
        want, mag, top, weights = test_shared_attn.formula(q.cpu().double(), pre.cpu().double(), torch.nan_to_num(tail.cpu().double()).reshape(slots, 2, -1, d), n.cpu(), scale)
        values = torch.cat([pre[:, 1].reshape(-1), torch.nan_to_num(tail[:, 1]).reshape(-1)]).cpu().double()
        assert ((out.cpu().double() - want).abs() <= test_shared_attn.tolerance(want, mag, top, values, prefix + slots, dt, d)).all()
        rel = 2 * top.max() * (d + 2) * 2.0 ** -23 + 2.0 ** -19
        assert ((w - before).cpu().double() - weights).abs().max() <= rel * weights.max() + w.max().item() * 2.0 ** -23
        count, rows, near, border = test_verify_drafts.by_rule(target.cpu(), draft.cpu(), tok.cpu(), None, u.cpu(), vocab, heat)
        if near > 2.0 ** -18 and border > 1e-11:
            assert np.array_equal(accepted.cpu().numpy(), count) and np.array_equal(chosen.cpu().numpy(), rows)
        passed += int(accepted.sum())
        # ---- what was not accepted leaves the tails, with its weights
        last = chosen.cpu().long()[torch.arange(batch), accepted.cpu().long()]
        n -= drafts - accepted
        w *= torch.arange(slots, device="cuda") < n[:, None, None]
        ring, old_w, old_n = tail.cpu(), w.cpu().numpy(), n.cpu().numpy()
        assert cuda.gehtp_kv_evict(a(tail), a(tail), a(w), a(w), a(n), a(n), a(kept), batch, kvh, d, slots, keep, sinks, recent, a(room[2]), room[2].numel(), stream) == 0
        torch.cuda.synchronize()
        for b in range(batch):
            cuts += int(old_n[b] > keep)
            for h in range(kvh):
                stay = test_kv_evict.rule(old_w[b, h], int(old_n[b]), keep, sinks, recent)
                assert kept[b, h, :len(stay)].tolist() == stay and int(n[b]) == len(stay)
                assert torch.equal(tail[:len(stay), :, b, h].cpu().view(torch.int16), ring[stay, :, b, h].view(torch.int16))
                assert np.array_equal(w[b, h].cpu().numpy(), np.concatenate([old_w[b, h, stay], np.zeros(slots - len(stay), np.float32)]))
    assert cuts > batch and passed > batch and cuda.gehtp_attn_shared_status() == 0
