"""The serving operators together, as a step uses them: q / k norm and rotation of a prompt batch with its cache rows, prompt
attention, the same for the drafted rows behind the cached prompt, shared attention over the cache, and verification of the
drafts; on one stream, captured and replayed. Each stage is checked in 64 bits from what the stage before left."""
import types

import numpy as np
import pytest

import serving_ref as ref
from test_gpu_serving_norm_verify import check_norm, check_verify
from test_gpu_serving_prompt import check as check_prompt
from test_gpu_serving_shared import check as check_shared

pytestmark = pytest.mark.gpu

F16, BF16 = 1, 30
H, KV, D, V = 8, 2, 128, 700
WIDE = (H + 2 * KV) * D
LENS, K = [210, 1, 37], [2, 0, 3, 1]  # prompts; drafts of each request, all of them behind the first prompt
POS = 512


class Step:
    def __init__(self, torch, mk, t, seed):
        dt = {F16: torch.float16, BF16: torch.bfloat16}[t]
        g = torch.Generator().manual_seed(seed)
        self.torch, self.mk, self.t, self.dt, self.g = torch, mk, t, dt, g
        self.n0, self.n1, self.R = sum(LENS), sum(K) + len(K), len(K)
        self.off = np.concatenate([[0], np.cumsum(LENS)])
        self.row_off = np.concatenate([[0], np.cumsum(np.asarray(K) + 1)])
        ang = torch.arange(POS)[:, None] / 10000.0 ** (torch.arange(D // 2)[None] * 2 / D)
        rows = self.n0
        kv_base, n_keys, at = [], [], []
        for k in K:  # a request's rows follow each other in the cache
            kv_base += [rows] * (k + 1)
            n_keys += list(range(1, k + 2))
            at += list(range(rows, rows + k + 1))
            rows += k + 1
        self.n_rows = rows
        i32 = lambda a: torch.as_tensor(np.asarray(a, np.int32)).cuda()  # noqa: E731
        self.pos0 = i32(np.concatenate([np.arange(n) for n in LENS]))
        self.at0 = i32(np.arange(self.n0))
        self.pos1 = i32(np.asarray(n_keys) - 1 + LENS[0])
        self.at1, self.kv_base, self.n_keys = i32(at), i32(kv_base), i32(n_keys)
        self.d_off, self.d_row_off = i32(self.off), i32(self.row_off)
        self.group = i32([0, self.n1])
        self.base, self.len = i32([0]), i32([LENS[0]])
        dev = lambda *s, dtype=dt: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        self.qw, self.kw = (dev(D, dtype=torch.float32) for _ in range(2))
        self.rope = torch.cat([ang.cos(), ang.sin()], 1).float().contiguous().cuda()
        self.in0, self.in1 = dev(self.n0, WIDE), dev(self.n1, WIDE)
        self.x0, self.q1 = dev(self.n0, WIDE), dev(self.n1, H * D)
        self.out0, self.out1 = dev(self.n0, H * D), dev(self.n1, H * D)
        self.kc, self.vc = (dev(KV, rows, D, dtype=torch.int8) for _ in range(2))
        self.ks, self.vs = (dev(KV, rows, dtype=torch.float32) for _ in range(2))
        self.head = dev(H * D, V)
        self.logits = dev(self.n1, V)
        self.nd = sum(K)
        self.draft = torch.zeros(self.nd, dtype=torch.int32, device="cuda")
        self.qp = dev(self.nd, V, dtype=torch.float32)
        self.temp = dev(self.R, dtype=torch.float32)
        self.u = dev(self.n1, dtype=torch.float64)
        self.n_acc, self.next = i32([0] * self.R), i32([0] * self.R)
        self.p = dev(self.nd, dtype=torch.float32)
        self.st = i32([0])
        self.ws_a = dev(mk.attention_shared_workspace(self.n1, H, KV, D, 1), dtype=torch.uint8)
        self.ws_v = dev(mk.verify_draft_workspace(self.n1, self.R, V), dtype=torch.uint8)

    def fill(self):
        torch, g = self.torch, self.g
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.in0.copy_(r(self.n0, WIDE))
        self.in1.copy_(r(self.n1, WIDE))
        self.qw.copy_(1 + 0.2 * r(D))
        self.kw.copy_(1 + 0.2 * r(D))
        self.head.copy_(r(H * D, V) * 0.5)
        q = torch.softmax(2 * r(self.nd, V), -1)
        self.qp.copy_(q)
        self.draft.copy_(torch.multinomial(q, 1, generator=g).flatten().int())
        self.temp.copy_(torch.tensor([0.7, 1.0, 0.0, 1.4]))
        self.u.copy_(torch.rand(self.n1, generator=g, dtype=torch.float64))
        for b in (self.kc, self.vc):
            b.fill_(99)
        for b in (self.ks, self.vs, self.out0, self.out1):
            b.fill_(float("nan"))

    def run(self, stream):
        mk, t, p = self.mk, self.t, lambda a: a.data_ptr()  # noqa: E731
        e = 2
        self.x0.copy_(self.in0)
        cache = (p(self.kc), p(self.vc), p(self.ks), p(self.vs), self.n_rows)
        mk.qk_norm_rope(t, p(self.x0), WIDE, self.n0, H, KV, D, p(self.qw), p(self.kw), 1e-6, p(self.rope), POS,
                        p(self.pos0), p(self.x0), WIDE, p(self.x0) + H * D * e, WIDE, *cache, p(self.at0), p(self.st),
                        stream)
        mk.attention_prompt(t, p(self.x0), WIDE, p(self.x0) + H * D * e, WIDE, p(self.x0) + (H + KV) * D * e, WIDE,
                            self.n0, len(LENS), p(self.d_off), H, KV, D, D ** -0.5, p(self.out0), H * D, p(self.st),
                            stream)
        mk.qk_norm_rope(t, p(self.in1), WIDE, self.n1, H, KV, D, p(self.qw), p(self.kw), 1e-6, p(self.rope), POS,
                        p(self.pos1), p(self.q1), H * D, 0, 0, *cache, p(self.at1), p(self.st), stream)
        mk.attention_shared(t, p(self.q1), H * D, self.n1, H, KV, D, D ** -0.5, *cache, 1, p(self.group), p(self.base),
                            p(self.len), p(self.kv_base), p(self.n_keys), 0, 0, 0, p(self.out1), H * D, p(self.ws_a),
                            self.ws_a.numel(), p(self.st), stream)
        self.torch.matmul(self.out1, self.head, out=self.logits)
        mk.verify_draft(t, p(self.logits), V, self.n1, V, self.R, p(self.d_row_off), p(self.draft), p(self.qp), V,
                        p(self.temp), p(self.u), p(self.n_acc), p(self.next), p(self.p), p(self.ws_v),
                        self.ws_v.numel(), p(self.st), stream)

    def check(self):
        torch, t = self.torch, self.t
        f = lambda a: a.float().cpu().numpy()  # noqa: E731
        assert int(self.st) == 0
        rope, qw, kw = f(self.rope), f(self.qw), f(self.kw)
        for src, pos, qs, ks in ((self.in0, self.pos0, f(self.x0)[:, :H * D], f(self.x0)[:, H * D:(H + KV) * D]),
                                 (self.in1, self.pos1, f(self.q1), None)):
            src, pos = f(src), pos.cpu().numpy()
            for i in range(len(src)):
                heads = src[i].reshape(-1, D)
                y, terms = ref.norm_rope(heads[:H], qw, 1e-6, rope[pos[i]])
                check_norm(torch, t, qs[i].reshape(-1, D), y, terms)
                if ks is not None:
                    y, terms = ref.norm_rope(heads[H:H + KV], kw, 1e-6, rope[pos[i]])
                    check_norm(torch, t, ks[i].reshape(-1, D), y, terms)
        check_prompt(torch, t, f(self.x0).astype(np.float64), self.off, f(self.out0), H, KV, D)
        b = types.SimpleNamespace(n=self.n1, k=self.kc.cpu().numpy(), v=self.vc.cpu().numpy(), ks=f(self.ks), vs=f(self.vs))
        assert np.isfinite(b.ks).all() and np.isfinite(b.vs).all()  # every row was written
        base, keys = self.kv_base.cpu().numpy(), self.n_keys.cpu().numpy()
        b.keys_of = lambda i: list(range(LENS[0])) + list(range(base[i], base[i] + keys[i]))
        check_shared(torch, t, b, self.q1, f(self.out1), H, KV, D)
        want = ref.verify(f(self.logits).astype(np.float64), self.row_off, self.draft.cpu().numpy(), f(self.qp),
                          f(self.temp), self.u.cpu().numpy())
        check_verify((self.n_acc.cpu().numpy(), self.next.cpu().numpy(), f(self.p), int(self.st)), want, self.nd)

    def results(self):
        return [a.clone() for a in (self.x0, self.out0, self.q1, self.out1, self.n_acc, self.next, self.p, self.kc, self.ks)]


@pytest.mark.parametrize("t", [F16, BF16])
def test_step(mk, torch_cuda, t):
    torch = torch_cuda
    s = Step(torch, mk, t, 3)
    for _ in range(3):
        s.fill()
        torch.cuda.synchronize()
        s.run(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        s.check()


def test_step_captured_beside_another(mk, torch_cuda):
    """Two steps with buffers of their own, captured, replayed at once on two streams with new inputs; a replay gives the
    bits of the queued calls."""
    torch = torch_cuda
    steps = [Step(torch, mk, t, 10 + t) for t in (F16, BF16)]
    streams = [torch.cuda.Stream() for _ in steps]
    graphs = []
    for s, q in zip(steps, streams):
        s.fill()
        torch.cuda.synchronize()
        with torch.cuda.stream(q):  # the matrix product's library sets itself up outside the capture
            s.run(q.cuda_stream)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=q):
            s.run(q.cuda_stream)
        graphs.append(g)
    for _ in range(4):
        for s in steps:
            s.fill()
        torch.cuda.synchronize()
        for g, q in zip(graphs, streams):
            with torch.cuda.stream(q):
                g.replay()
        torch.cuda.synchronize()
        for s in steps:
            s.check()
            first = s.results()
            s.run(torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            for a, b in zip(first, s.results()):
                assert torch.equal(a, b)


def test_offsets_beyond_32_bits(mk, torch_cuda):
    """Buffers of more than 2^32 bytes and 2^31 elements, used at their far ends."""
    torch = torch_cuda
    d = lambda a, dt=torch.int32: torch.as_tensor(np.asarray(a)).to(dt).cuda()  # noqa: E731
    st, g = d([0]), torch.Generator().manual_seed(1)
    # rows 2^22 elements apart, 600 of them: prompt attention and the norm in place, then its cache rows far out
    ld, n, rows = 1 << 22, 600, 18_000_000
    x = torch.empty(n * ld, dtype=torch.bfloat16, device="cuda").view(n, ld)
    x[:, :WIDE] = torch.randn(n, WIDE, generator=g).bfloat16().cuda()
    kc, vc = (torch.empty(KV, rows, D, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(KV, rows, dtype=torch.float32, device="cuda") for _ in range(2))
    assert x.numel() > 2 ** 31 and kc.numel() > 2 ** 32
    raw = x[:, :WIDE].float().cpu().numpy()
    ang = torch.rand(n, D // 2, generator=g) * 6
    rope = torch.cat([ang.cos(), ang.sin()], 1).contiguous().cuda()
    w, pos, at = torch.ones(D, device="cuda"), d(np.arange(n)), d(np.arange(rows - n, rows))
    e = 2
    mk.qk_norm_rope(BF16, x.data_ptr(), ld, n, H, KV, D, w.data_ptr(), w.data_ptr(), 1e-6, rope.data_ptr(), n,
                    pos.data_ptr(), x.data_ptr(), ld, x.data_ptr() + H * D * e, ld, kc.data_ptr(), vc.data_ptr(),
                    ks.data_ptr(), vs.data_ptr(), rows, at.data_ptr(), st.data_ptr())
    torch.cuda.synchronize()
    got = x[:, :WIDE].float().cpu().numpy()
    for i in (0, n - 1):
        y, terms = ref.norm_rope(raw[i].reshape(-1, D)[:H + KV], np.ones(D), 1e-6, rope[i].cpu().numpy())
        check_norm(torch, BF16, got[i].reshape(-1, D)[:H + KV], y, terms)
        held = vc[:, rows - n + i].cpu().numpy() * vs[:, rows - n + i].cpu().numpy()[:, None]
        v = raw[i].reshape(-1, D)[H + KV:]
        assert np.all(np.abs(held - v) <= np.abs(v).max(-1, keepdims=True) / 127 * 0.5001)
    out = x[:, WIDE:WIDE + H * D]
    off = d([0, 300, 600])
    mk.attention_prompt(BF16, x.data_ptr(), ld, x.data_ptr() + H * D * e, ld, x.data_ptr() + (H + KV) * D * e, ld, n, 2,
                        off.data_ptr(), H, KV, D, D ** -0.5, out.data_ptr(), ld, st.data_ptr())
    torch.cuda.synchronize()
    check_prompt(torch, BF16, got.astype(np.float64), off.cpu().numpy(), out.float().cpu().numpy(), H, KV, D)
    # the far rows as a prefix of 500 and own rows behind it
    tok = 4
    b = types.SimpleNamespace(n=tok, k=kc[:, rows - n:].cpu().numpy(), v=vc[:, rows - n:].cpu().numpy(),
                              ks=ks[:, rows - n:].cpu().numpy(), vs=vs[:, rows - n:].cpu().numpy())
    b.keys_of = lambda i: list(range(500 + i)) + [n - 1]
    args = [d(a) for a in ([0, tok], [rows - n], [500], [rows - n + 500] * tok, range(tok), range(tok + 1), [99] * tok)]
    y = torch.empty(tok, H * D, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(mk.attention_shared_workspace(tok, H, KV, D, 1), dtype=torch.uint8, device="cuda")
    mk.attention_shared(BF16, x.data_ptr() + (n - tok) * ld * e, ld, tok, H, KV, D, D ** -0.5, kc.data_ptr(),
                        vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), rows, 1, *[a.data_ptr() for a in args], tok,
                        y.data_ptr(), H * D, ws.data_ptr(), ws.numel(), st.data_ptr())
    torch.cuda.synchronize()
    check_shared(torch, BF16, b, x[n - tok:, :H * D], y.float().cpu().numpy(), H, KV, D)
    # logits rows that far apart
    lg = x[:, :V]
    lg[n - 3:] = (torch.randn(3, V, generator=g) * 3).bfloat16().cuda()
    row_off, draft = d([0, 597, 600]), d(np.arange(598) % V)
    u, temp = torch.rand(n, generator=g, dtype=torch.float64).cuda(), torch.ones(2, device="cuda")
    n_acc, nxt, p = d([0, 0]), d([0, 0]), torch.empty(598, device="cuda")
    wv = torch.empty(mk.verify_draft_workspace(n, 2, V), dtype=torch.uint8, device="cuda")
    mk.verify_draft(BF16, x.data_ptr(), ld, n, V, 2, row_off.data_ptr(), draft.data_ptr(), 0, 0, temp.data_ptr(),
                    u.data_ptr(), n_acc.data_ptr(), nxt.data_ptr(), p.data_ptr(), wv.data_ptr(), wv.numel(), st.data_ptr())
    torch.cuda.synchronize()
    want = ref.verify(lg.float().cpu().numpy().astype(np.float64), [0, 597, 600], draft.cpu().numpy(), None,
                      [1.0, 1.0], u.cpu().numpy())
    check_verify((n_acc.cpu().numpy(), nxt.cpu().numpy(), p.cpu().numpy(), int(st)), want, 598)


def test_steps_from_several_host_threads(mk, torch_cuda):
    """Four host threads at once, each with a step and a stream of its own: the results are those of the calls made alone."""
    import threading
    torch = torch_cuda
    steps = [Step(torch, mk, (F16, BF16)[i % 2], 30 + i) for i in range(4)]
    streams = [torch.cuda.Stream() for _ in steps]
    for s in steps:
        s.fill()
        s.run(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = [s.results() for s in steps]
    failed = []

    def work(s, q):
        try:
            with torch.cuda.stream(q):
                for _ in range(20):
                    s.run(q.cuda_stream)
        except Exception as e:  # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=work, args=a) for a in zip(steps, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for s, w in zip(steps, want):
        assert all(torch.equal(a, b) for a, b in zip(s.results(), w))
