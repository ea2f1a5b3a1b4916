"""mk_qk_norm_rope and mk_verify_draft on the GPU against plain 64-bit forms."""
import numpy as np
import pytest

import serving_ref as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 30


def torch_type(torch, t):
    return {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[t]


def half_step(torch, t):
    return torch.finfo(torch_type(torch, t)).eps / 2


def host(x):
    return x.detach().float().cpu().numpy()


# ---------------- q / k norm and rotation ----------------
# Error of an output beside its two terms a, b (|a| + |b| is what the reference returns as its second value): the sum of D
# squares is 8 additions in a lane and at most 5 between lanes, 13 roundings whose effect the square root halves; mean and
# eps 2 more (halved); rsqrt is good to 2 steps of 2^-23 (4 half steps); x r w two roundings; the rotation two products and
# one sum. At most 7.5 + 4 + 2 + 3 < 17 half steps of 2^-24 on |a| + |b|, then the rounding to the type.
NORM_STEPS = 17 * 2.0 ** -24


def norm_inputs(torch, t, n, H, KV, D, ld, offset, seed):
    g = torch.Generator().manual_seed(seed)
    buf = torch.full((offset + n * ld,), float("nan"))
    x = buf[offset:].view(n, ld)
    x[:, :(H + 2 * KV) * D] = torch.randn(n, (H + 2 * KV) * D, generator=g) * 1.7
    buf = buf.to(torch_type(torch, t)).cuda()
    return buf, buf[offset:].view(n, ld)


def check_norm(torch, t, got, want, terms):
    tol = NORM_STEPS * terms + half_step(torch, t) * np.abs(want) + 2.0 ** -25 * (t == F16)
    # fp16 results below 2^-14 are subnormal: half a step is 2^-25 there
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.abs(got - want).max(), np.argwhere(bad)[:3])


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("n,H,KV,D,pad,offset", [(1, 4, 2, 128, 0, 0), (3, 5, 1, 64, 4, 0), (17, 32, 8, 128, 8, 4),
                                                 (2, 7, 3, 256, 0, 0), (5, 3, 2, 128, 1, 0), (4, 2, 1, 64, 3, 3),
                                                 (130, 16, 8, 128, 0, 0)])
def test_norm_rope(mk, torch_cuda, t, n, H, KV, D, pad, offset):
    torch = torch_cuda
    ld = (H + 2 * KV) * D + pad
    buf, x = norm_inputs(torch, t, n, H, KV, D, ld, offset, 7 * n + D)
    g = torch.Generator().manual_seed(3)
    qw, kw = (1 + 0.3 * torch.randn(D, generator=g) for _ in range(2))
    n_pos = 50
    ang = torch.rand(n_pos, D // 2, generator=g) * 6
    rope = torch.cat([ang.cos(), ang.sin()], 1).contiguous()
    pos = torch.randint(0, n_pos, (n,), generator=g).int()
    if n > 2:
        pos[1] = -1  # padding
    q_ld, k_ld = H * D + 4, KV * D + pad
    q = torch.full((n, q_ld), -7.0, dtype=x.dtype, device="cuda")
    k = torch.full((n, k_ld), -7.0, dtype=x.dtype, device="cuda")
    d = [v.cuda() for v in (qw, kw, rope, pos)]
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    mk.qk_norm_rope(t, x.data_ptr(), ld, n, H, KV, D, d[0].data_ptr(), d[1].data_ptr(), 1e-6, d[2].data_ptr(), n_pos,
                    d[3].data_ptr(), q.data_ptr(), q_ld, k.data_ptr(), k_ld, dev_status=st.data_ptr())
    torch.cuda.synchronize()
    assert int(st) == 0
    xs, qs, ks = host(x), host(q), host(k)
    for i in range(n):
        p = int(pos[i])
        if p < 0:
            assert (qs[i] == -7).all() and (ks[i] == -7).all()
            continue
        heads = xs[i, :(H + 2 * KV) * D].reshape(-1, D)
        for lo, m, w, got in ((0, H, qw, qs[i, :H * D]), (H, KV, kw, ks[i, :KV * D])):
            want, terms = ref.norm_rope(heads[lo:lo + m], w.numpy(), 1e-6, rope[p].numpy())
            check_norm(torch, t, got.reshape(m, D), want, terms)
        assert (qs[i, H * D:] == -7).all() and (ks[i, KV * D:] == -7).all()


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_norm_rope_in_place_with_cache(mk, torch_cuda, t, D):
    """In place, with cache rows in any order, rows left alone (kv_at < 0), a zero head and a status for a row outside."""
    torch = torch_cuda
    n, H, KV, rows = 9, 6, 3, 20
    ld = (H + 2 * KV) * D
    _, x = norm_inputs(torch, t, n, H, KV, D, ld, 0, 11)
    x[2, (H + KV) * D:(H + KV + 1) * D] = 0  # a value head of zeros: scale 0
    before = host(x).copy()
    g = torch.Generator().manual_seed(5)
    qw, kw = (1 + 0.3 * torch.randn(D, generator=g) for _ in range(2))
    ang = torch.rand(n, D // 2, generator=g) * 6
    rope = torch.cat([ang.cos(), ang.sin()], 1).contiguous()
    pos = torch.arange(n).int()
    at = torch.tensor([5, 0, 19, -1, 7, rows, 3, 11, 1]).int()
    d = [v.cuda() for v in (qw, kw, rope, pos, at)]
    kc, vc = (torch.full((KV, rows, D), 99, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((KV, rows), -1.0, device="cuda") for _ in range(2))
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    mk.qk_norm_rope(t, x.data_ptr(), ld, n, H, KV, D, d[0].data_ptr(), d[1].data_ptr(), 1e-6, d[2].data_ptr(), n,
                    d[3].data_ptr(), x.data_ptr(), ld, x.data_ptr() + H * D * x.element_size(), ld, kc.data_ptr(),
                    vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), rows, d[4].data_ptr(), st.data_ptr())
    torch.cuda.synchronize()
    assert int(st) == mk.MK_ERR_ARG  # token 5's row is one past the cache
    after = host(x)
    held = {name: (a.cpu().numpy(), b.cpu().numpy()) for name, a, b in (("k", kc, ks), ("v", vc, vs))}
    written = set()
    for i in range(n):
        heads = before[i].reshape(-1, D)
        want = []
        for lo, m, w in ((0, H, qw), (H, KV, kw)):
            y, terms = ref.norm_rope(heads[lo:lo + m], w.numpy(), 1e-6, rope[i].numpy())
            check_norm(torch, t, after[i].reshape(-1, D)[lo:lo + m], y, terms)
            want.append(y)
        assert np.array_equal(after[i].reshape(-1, D)[H + KV:], heads[H + KV:])  # values are left as they were
        r = int(at[i])
        if not 0 <= r < rows:
            continue
        written.add(r)
        for name, y in (("k", want[1]), ("v", heads[H + KV:].astype(np.float64))):
            q8, sc = held[name]
            amax = np.abs(y).max(-1)
            # scale: amax / 127 from values that carry NORM_STEPS; a held value is off by half a step of it and that error
            slack = 2 * NORM_STEPS * 2 * np.abs(y).max() * 1.5
            assert np.all(np.abs(sc[:, r] - amax / 127) <= slack / 127 + 2.0 ** -23 * amax / 127)
            err = np.abs(q8[:, r].astype(np.float64) * sc[:, r][:, None].astype(np.float64) - y)
            assert np.all(err <= 0.5 * sc[:, r][:, None] * (1 + 2.0 ** -16) + slack), (name, err.max())
    for q8, sc in held.values():
        for r in range(rows):
            if r not in written:
                assert (q8[:, r] == 99).all() and (sc[:, r] == -1).all()


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("H,KV,D,cache,inplace", [(32, 8, 128, True, False), (32, 8, 128, False, True), (24, 8, 64, True, True),
                                                  (7, 3, 256, True, False), (64, 8, 64, False, False), (5, 1, 64, True, False)])
def test_norm_rope_large_batches(mk, torch_cuda, t, H, KV, D, cache, inplace):
    """A large batch gives the bits that its tokens give in small ones, padding, refused indexes and untouched rows among them;
    the first and last tokens against the 64-bit form."""
    torch = torch_cuda
    n, rows, n_pos = 4001, 5000, 500
    ld = (H + 2 * KV) * D + 16
    _, x = norm_inputs(torch, t, n, H, KV, D, ld, 0, 3)
    before = x.clone()
    g = torch.Generator().manual_seed(8)
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).cuda() for _ in range(2))
    ang = torch.rand(n_pos, D // 2, generator=g) * 6
    rope = torch.cat([ang.cos(), ang.sin()], 1).contiguous().cuda()
    pos = torch.randint(0, n_pos, (n,), generator=g).int()
    pos[[5, 700, 3999]] = torch.tensor([-1, n_pos, -7]).int()
    at = torch.randperm(rows, generator=g)[:n].int()
    at[[6, 1700]] = torch.tensor([-1, rows]).int()
    pos, at = pos.cuda(), at.cuda()

    def call(step):
        src = before.clone()
        q, k = (torch.full((n, w * D), 7.0, dtype=x.dtype, device="cuda") for w in (H, KV))
        qp, kp, q_ld, k_ld = q.data_ptr(), k.data_ptr(), H * D, KV * D
        e = src.element_size()
        if inplace:
            qp, kp, q_ld, k_ld = src.data_ptr(), src.data_ptr() + H * D * e, ld, ld
        kc, vc = (torch.full((KV, rows, D), 99, dtype=torch.int8, device="cuda") for _ in range(2))
        ks, vs = (torch.full((KV, rows), -1.0, device="cuda") for _ in range(2))
        st = torch.zeros(1, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        for lo in range(0, n, step):
            held = (kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), rows, at.data_ptr() + 4 * lo) if cache else ()
            mk.qk_norm_rope(t, src.data_ptr() + lo * ld * e, ld, min(step, n - lo), H, KV, D, qw.data_ptr(), kw.data_ptr(),
                            1e-6, rope.data_ptr(), n_pos, pos.data_ptr() + 4 * lo, qp + lo * q_ld * e, q_ld,
                            kp + lo * k_ld * e, k_ld, *held, dev_status=st.data_ptr())
        torch.cuda.synchronize()
        assert int(st) == mk.MK_ERR_ARG
        if inplace:
            q, k = src[:, :H * D], src[:, H * D:(H + KV) * D]
        return [a.contiguous().view(torch.uint8) for a in (src, q, k, kc, vc, ks, vs)] + [host(q), host(k)]

    large, small = call(n), call(97)
    for a, b in zip(large[:7], small[:7]):
        assert torch.equal(a, b)
    for i in (0, n - 1):
        heads = host(before[i, :(H + KV) * D]).reshape(-1, D)
        for got, lo, m, w in ((large[7], 0, H, qw), (large[8], H, KV, kw)):
            y, terms = ref.norm_rope(heads[lo:lo + m], host(w), 1e-6, host(rope[int(pos[i])]))
            check_norm(torch, t, got[i].reshape(-1, D), y, terms)


# ---------------- verification ----------------
# p of a draft: its own exponential is in 64 bits, the row's sum is of 32-bit exponentials 2^t: t carries two roundings
# (2^-23 |t| ln 2 relative), entries below 2^-40 of the maximum weigh nothing, exp2f is good to 2 steps, sums and the
# block's rescaling add at most 20 half steps: (40 ln 2 + 2 + 10 + 1) 2^-23 < 42 * 2^-23.
P_REL = 42 * 2.0 ** -23


def verify_call(mk, torch, t, logits, ld, row_off, draft, q, q_ld, temp, u, V, R, stream=0, ws=None):
    n_acc, nxt = (torch.full((R,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    p = torch.full((max(len(draft), 1),), -9.0, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows = logits.shape[0]
    if ws is None:
        ws = torch.empty(mk.verify_draft_workspace(rows, R, V), dtype=torch.uint8, device="cuda")
    d = [torch.as_tensor(a).cuda() for a in (np.asarray(row_off, np.int32), np.asarray(list(draft) or [0], np.int32),
                                             np.asarray(temp, np.float32), np.asarray(u, np.float64))]
    mk.verify_draft(t, logits.data_ptr(), ld, rows, V, R, d[0].data_ptr(), d[1].data_ptr(),
                    q.data_ptr() if q is not None else 0, q_ld, d[2].data_ptr(), d[3].data_ptr(), n_acc.data_ptr(),
                    nxt.data_ptr(), p.data_ptr(), ws.data_ptr(), ws.numel(), st.data_ptr(), stream)
    torch.cuda.synchronize()
    return n_acc.cpu().numpy(), nxt.cpu().numpy(), p.cpu().numpy(), int(st)


def as64(logits):
    x = logits.float().cpu().numpy().astype(np.float64)
    return np.where(np.isnan(x), -np.inf, x)


def check_verify(got, want, nd):
    assert np.array_equal(got[0], want[0]), (got[0], want[0])
    assert np.array_equal(got[1], want[1]), (got[1], want[1])
    if nd:
        assert np.all(np.abs(got[2] - want[2]) <= P_REL * want[2] + 2.0 ** -126)
    assert got[3] == 0


def drafts_near(torch, logits, rows, temp_rows, g):
    V = logits.shape[1]
    x = logits[rows].float().cpu()
    q = torch.softmax((x + 0.7 * torch.randn(x.shape, generator=g)) / torch.as_tensor(temp_rows)[:, None].clamp(min=0.5), -1)
    q = torch.nan_to_num(q)
    return q, torch.multinomial(q + 1e-30, 1, generator=g).flatten().numpy()


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("V,kk,with_q,pad", [(1, [0, 2], True, 0), (7, [3, 0, 1], True, 1), (33, [4], False, 0),
                                             (1000, [2, 5, 0, 1], True, 0), (4096, [3, 3], False, 3),
                                             (5003, [8, 1], True, 5), (40001, [2, 0, 6], True, 0),
                                             (151936, [4, 2], True, 0), (151936, [1, 3], False, 0)])
def test_verify(mk, torch_cuda, t, V, kk, with_q, pad):
    torch = torch_cuda
    R, off = len(kk), np.concatenate([[0], np.cumsum(np.asarray(kk) + 1)])
    rows = int(off[-1])
    for seed in range(4):
        g = torch.Generator().manual_seed(seed * 100 + V)
        logits = torch.zeros(rows, V + pad)
        logits[:, :V] = torch.randn(rows, V, generator=g) * (0.3 if seed == 3 else 3)
        logits = logits.to(torch_type(torch, t)).cuda()
        temp = np.where(np.arange(R) % 3 == 1, 0.0, 0.5 + 0.3 * np.arange(R)).astype(np.float32)
        dr = np.concatenate([np.arange(off[r], off[r + 1] - 1) for r in range(R)]).astype(np.int64)
        of = np.concatenate([np.full(kk[r], r) for r in range(R)]).astype(np.int64)
        q, draft = drafts_near(torch, logits[:, :V], dr, temp[of], g) if len(dr) else (torch.zeros(1, V), np.zeros(0))
        u = torch.rand(rows, generator=g, dtype=torch.float64).numpy()
        qd = None
        if with_q:
            qd = torch.zeros(max(len(dr), 1), V + 2)
            qd[:, :V] = q
            qd = qd.cuda()
        got = verify_call(mk, torch, t, logits, V + pad, off, draft, qd, V + 2, temp, u, V, R)
        want = ref.verify(as64(logits[:, :V]), off, draft, q.numpy() if with_q else None, temp, u)
        check_verify(got, want, len(draft))


def test_verify_edges(mk, torch_cuda):
    """Masked tokens, rows without a distribution, drafts outside the vocabulary, q of 0, p <= q everywhere, uniforms 0
    and almost 1, ties of the greedy maximum, tiny and infinite temperatures."""
    torch = torch_cuda
    V = 300
    g = torch.Generator().manual_seed(1)
    base = torch.randn(40, V, generator=g) * 2
    rows, off, draft, temp, u, q, exp = [], [0], [], [], [], [], []
    inf, nan = float("inf"), float("nan")

    def request(lg, dr, tm, us, qs):
        rows.extend(lg)
        off.append(off[-1] + len(lg))
        draft.extend(dr)
        temp.append(tm)
        u.extend(us)
        q.extend(qs)

    soft = lambda x, tm: torch.softmax(x.double() / tm, -1).float()  # noqa: E731
    masked = base[0].clone()
    masked[:290] = -inf
    masked[295] = nan
    request([masked, masked], [3], 1.0, [0.0, 0.999999999], [soft(base[1], 1.0)])            # a masked draft: refused
    request([torch.full((V,), -inf)], [], 1.0, [0.5], [])                                     # nothing to draw from
    request([base[2], torch.full((V,), nan)], [5], 1.0, [0.0, 0.5], [soft(base[2], 1.0)])     # kept, then nothing
    request([torch.full((V,), inf), base[3]], [5], 1.0, [0.5, 0.5], [soft(base[3], 1.0)])     # no distribution: not kept
    request([base[4], base[5]], [V], 1.0, [0.0, 0.3], [soft(base[4], 1.0)])                   # draft past the vocabulary
    request([base[6], base[7]], [-1], 1.0, [0.0, 0.3], [soft(base[6], 1.0)])
    zero = soft(base[8], 1.0)
    zero[9] = 0
    request([base[8], base[9]], [9], 1.0, [0.0, 0.7], [zero])                                 # q(d) = 0: refused
    p = soft(base[10], 1.0)
    request([base[10], base[11]], [int(p.argmin())], 1.0, [0.9999999, 0.6], [p * 1.5 + 1e-6])  # p <= q: draw from p
    tie = base[12].clone()
    tie[[17, 40, 299]] = 50.0
    request([tie, tie], [17], 0.0, [0.5, 0.5], [soft(tie, 1.0)])                              # greedy: lowest index
    request([tie, tie], [40], -1.0, [0.5, 0.5], [soft(tie, 1.0)])                             # not the lowest: refused
    request([base[13]], [], 1.0, [0.0], [])                                                   # u = 0: first token
    request([base[14]], [], 1.0, [1.0 - 2.0 ** -53], [])                                      # u almost 1: last token
    request([base[15]], [], 1e-3, [0.5], [])                                                  # one token left
    request([base[16]], [], inf, [0.5], [])                                                   # every token alike
    request([masked], [], inf, [0.99], [])
    request([base[17]], [], 1e-42, [0.5], [])
    R = len(temp)
    lg = torch.stack(rows).cuda()
    qd = torch.stack(q).cuda()
    got = verify_call(mk, torch, F32, lg, V, off, draft, qd, V, temp, u, V, R)
    with np.errstate(all="ignore"):
        x = as64(lg)
        tm = np.asarray(temp, np.float32).astype(np.float64)
        fix = x.copy()
        for r in range(R):
            if np.isinf(tm[r]):  # the limit: 0 where the token is there, -inf where it is masked
                fix[off[r]:off[r + 1]] = np.where(np.isfinite(x[off[r]:off[r + 1]]), 0.0, -np.inf)
        t2 = np.where(np.isinf(tm), 1.0, tm)
        want = ref.verify(fix, off, draft, qd.cpu().numpy(), t2, u)
    check_verify(got, want, len(draft))
    assert got[1][1] == -1 and got[0][2] == 1 and got[1][2] == -1 and got[0][3] == 0 and got[1][3] == -1
    assert got[0][8] == 1 and got[1][8] == 17 and got[0][9] == 0 and got[1][10] == 0 and got[1][11] == V - 1
    assert got[1][0] >= 290 and got[1][14] >= 290 and got[1][14] != 295


@pytest.mark.parametrize("temp", [float("inf"), 3e38, 1e-38])
def test_verify_extreme_temperatures(mk, torch_cuda, temp):
    """Towards infinity every token that can be drawn weighs the same, towards 0 the maximum takes all."""
    torch = torch_cuda
    V = 5003
    logits = torch.randn(3, V, generator=torch.Generator().manual_seed(1)).cuda()
    logits[:, 1::2] = -float("inf")
    top = int(logits[0].argmax())
    some = (V + 1) // 2
    got = verify_call(mk, torch, F32, logits, V, [0, 2, 3], [top], None, 0, [temp, temp], [0.0, 0.5, 0.25], V, 2)
    assert got[3] == 0 and list(got[0]) == [1, 0]
    want = [int(logits[1].argmax()), int(logits[2].argmax())]
    if temp > 1:
        assert abs(got[2][0] - 1 / some) <= P_REL / some
        want = [2 * (-(-some // 2) - 1), 2 * (-(-some // 4) - 1)]  # the first whose rank reaches u x some
    else:
        assert got[2][0] == 1
    assert list(got[1]) == want


def test_verify_bad_tables(mk, torch_cuda):
    """Offsets that run backwards, past the rows or below zero: those requests give (0, -1) and the status, the others
    their results."""
    torch = torch_cuda
    V, rows, R = 64, 6, 3
    g = torch.Generator().manual_seed(2)
    lg = (torch.randn(rows, V, generator=g) * 2).cuda()
    u = torch.rand(rows, generator=g, dtype=torch.float64).numpy()
    draft = [1, 2, 3]
    good = verify_call(mk, torch, F32, lg, V, [0, 2, 4, 6], draft, None, 0, [1.0] * 3, u, V, R)
    assert good[3] == 0
    for off, bad in (([0, 2, 4, 7], [2]), ([0, 2, 2, 6], [1]), ([-1, 2, 4, 6], [0]), ([0, 2, 9, 6], [1, 2])):
        got = verify_call(mk, torch, F32, lg, V, off, draft, None, 0, [1.0] * 3, u, V, R)
        assert got[3] == mk.MK_ERR_ARG, off
        for r in range(R):
            if r in bad:
                assert got[0][r] == 0 and got[1][r] == -1, (off, r, got)
            elif off[r:r + 2] == [2 * r, 2 * r + 2]:
                assert got[0][r] == good[0][r] and got[1][r] == good[1][r], (off, r)


def test_verify_many_requests_and_graph(mk, torch_cuda):
    """More requests than a block has threads, ragged, on a stream of its own; the same call captured and replayed with
    other logits in the same buffers."""
    torch = torch_cuda
    R, V = 300, 513
    kk = [(r * 7) % 4 for r in range(R)]
    off = np.concatenate([[0], np.cumsum(np.asarray(kk) + 1)])
    rows = int(off[-1])
    g = torch.Generator().manual_seed(9)
    temp = np.where(np.arange(R) % 5 == 4, 0.0, 0.8).astype(np.float32)
    dr = np.concatenate([np.arange(off[r], off[r + 1] - 1) for r in range(R)]).astype(np.int64)
    of = np.concatenate([np.full(kk[r], r) for r in range(R)]).astype(np.int64)
    first = torch.randn(rows, V, generator=g) * 2
    q, draft = drafts_near(torch, first, dr, temp[of], g)
    u = torch.rand(rows, generator=g, dtype=torch.float64).numpy()
    lg, qd = first.to(torch.bfloat16).cuda(), q.cuda()
    s = torch.cuda.Stream()
    ws = torch.empty(mk.verify_draft_workspace(rows, R, V), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    got = verify_call(mk, torch, BF16, lg, V, off, draft, qd, V, temp, u, V, R, stream=s.cuda_stream, ws=ws)
    check_verify(got, ref.verify(as64(lg), off, draft, q.numpy(), temp, u), len(draft))
    n_acc, nxt = (torch.zeros(R, dtype=torch.int32, device="cuda") for _ in range(2))
    p = torch.zeros(len(draft), device="cuda")
    d = [torch.as_tensor(a).cuda() for a in (np.asarray(off, np.int32), np.asarray(draft, np.int32), temp, u)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mk.verify_draft(BF16, lg.data_ptr(), V, rows, V, R, d[0].data_ptr(), d[1].data_ptr(), qd.data_ptr(), V,
                        d[2].data_ptr(), d[3].data_ptr(), n_acc.data_ptr(), nxt.data_ptr(), p.data_ptr(), ws.data_ptr(),
                        ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
    for k in range(2):
        lg.copy_((torch.randn(rows, V, generator=g) * 2 + first).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        want = ref.verify(as64(lg), off, draft, q.numpy(), temp, u)
        check_verify((n_acc.cpu().numpy(), nxt.cpu().numpy(), p.cpu().numpy(), 0), want, len(draft))


@pytest.mark.parametrize("R,rows,off,same,bad", [
    (3, 6, [0, 9, 4, 6], [0, 2, 4, 6], [0, 1]),    # the first two leave the rows, the third stands by itself
    (3, 6, [0, 2, -1, 6], [0, 2, 4, 6], [1, 2]),   # rows of the first behind which two bad ends lie
    (3, 6, [3, 1, 4, 6], [0, 1, 4, 6], [0]),
    (3, 8, [2, 6, 3, 7], [2, 6, 7, 8], [1, 2]),    # the third over the first's rows
    (4, 9, [0, 3, 3, 6, 9], [0, 3, 4, 6, 9], [1, 2])])  # an empty request: the third's drafts would be the first's
def test_verify_bad_tables_leave_the_others(mk, torch_cuda, R, rows, off, same, bad):
    """Requests whose own rows are right keep their results, each with its own temperature, whatever stands beside them;
    a request over an earlier one's rows or drafts is refused. `same`: a right table in which the others have the same rows."""
    torch = torch_cuda
    V = 500
    for seed in range(6):
        g = torch.Generator().manual_seed(seed)
        lg = (torch.randn(rows, V, generator=g) * 2).cuda()
        u = torch.rand(rows, generator=g, dtype=torch.float64).numpy()
        draft = torch.randint(0, V, (rows - R,), generator=g).numpy()
        temp = [[1.0, 0.0, 0.7, 2.5], [0.0, 0.9, 1.3, 0.0], [3.0, 0.5, 0.0, 1.0]][seed % 3][:R]
        good = verify_call(mk, torch, F32, lg, V, same, draft, None, 0, temp, u, V, R)
        assert good[3] == 0
        got = verify_call(mk, torch, F32, lg, V, off, draft, None, 0, temp, u, V, R)
        assert got[3] == mk.MK_ERR_ARG
        for r in range(R):
            if r in bad:
                assert got[0][r] == 0 and got[1][r] == -1, (seed, r, got)
            else:
                assert got[0][r] == good[0][r] and got[1][r] == good[1][r], (seed, r, got, good)
                js = slice(off[r] - r, off[r + 1] - 1 - r)
                assert np.array_equal(got[2][js], good[2][js]), (seed, r)


def test_verify_residual_of_one_rounding(mk, torch_cuda):
    """One entry of the residual is above 0, by less than a rounding of the row's sum: found by trying temperatures until
    p - q had that sign for the sum of the 384 chunks' shares taken 256 at a time, and the other one taken 512 at a time. The
    token drawn is that entry, since the sum behind the residual's total is also the one behind the draw."""
    torch = torch_cuda
    chunks, size, temp, seed = 384, 4096, 1.88917732, 2076039816
    V = chunks * size
    lg = torch.full((2, V), -float("inf"))
    s, classes = 2 * seed + 1, []
    for i in range(chunks):  # one token a chunk, 0, 1, 2 or 4 below the first
        s = (s * 6364136223846793005 + 1442695040888963407) % 2 ** 64
        classes.append(0 if i == 0 else (s >> 40) & 3)
        lg[:, i * size + 17] = -[0.0, 1.0, 2.0, 4.0][classes[-1]]
    token = classes.index(3) * size + 17
    q = torch.ones(1, V)
    q[0, token] = 0.000591546181
    got = verify_call(mk, torch, F32, lg.cuda(), V, [0, 2], [17], q.cuda(), V, [temp], [0.99, 0.5], V, 1)
    assert got[0][0] == 0 and got[1][0] == token and got[3] == 0, got


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("V,with_q", [(700, True), (30011, True), (151936, False)])
def test_verify_at_the_border(mk, torch_cuda, t, V, with_q):
    """u q(d) a part in 10^11 below and above p(d): the acceptance is that of the 64-bit rule, one draft or several in a
    row (both sides' sums are good to some 10^-13)."""
    torch = torch_cuda
    R, K = 24, 3
    g = torch.Generator().manual_seed(V)
    lg = (torch.randn(R * (K + 1), V, generator=g) * 1.5).to(torch_type(torch, t)).cuda()
    x = as64(lg)
    temp = (0.6 + 0.05 * np.arange(R)).astype(np.float32)
    off = np.arange(R + 1) * (K + 1)
    draft, u = np.zeros(R * K, np.int64), np.full(R * (K + 1), 0.4)
    q = np.full((R * K, V), 0.5 / V, np.float32)
    stop = [r % (K + 1) for r in range(R)]  # the draft that is refused; K: none
    for r in range(R):
        for i in range(K):
            p = ref.softmax(x[off[r] + i] / np.float64(temp[r]))
            d = int(np.argsort(-p)[3 + i])
            draft[r * K + i] = d
            q[r * K + i, d] = 1.25 * p[d]
            qd = float(q[r * K + i, d]) if with_q else 1.0
            u[off[r] + i] = p[d] / qd * (1 + 1e-11 if i >= stop[r] else 1 - 1e-11)
    qd = torch.as_tensor(q).cuda() if with_q else None
    got = verify_call(mk, torch, t, lg, V, off, draft, qd, V, temp, u, V, R)
    want = ref.verify(x, off, draft, q if with_q else None, temp, u)
    assert list(want[0]) == stop
    check_verify(got, want, len(draft))
