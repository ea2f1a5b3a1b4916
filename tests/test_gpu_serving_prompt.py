"""mk_attention_prompt on the GPU against softmax attention in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F16, BF16 = 1, 30

# Error of an output beside A = sum_j w_j |v_j| (weights w of the exact softmax), h = half a step of the type:
#   weights are rounded to the type: h on each;
#   fp32: the score is a sum of D products (D 2^-24 of sum |q k| scale, below 2^-17 x the spread of scores for these
#   inputs), its exponent two roundings, ex2 2 steps, the row's sum and the product's sum up to 2^-24 per key:
#   together below (|s| 2^-16 + L 2^-24 + 2^-20) A with |s| <= 24 here, so 2^-11 A covers it;
# then the rounding of the output: h |out|.
FP32_PART = 2.0 ** -11


def tt(torch, t):
    return {F16: torch.float16, BF16: torch.bfloat16}[t]


def exact(q, k, v, scale):
    """q [L, H, D], k, v [L, KV, D] float64 -> out, A (see above)."""
    L, H, D = q.shape
    G = H // k.shape[1]
    out, mag = np.zeros((L, H, D)), np.zeros((L, H, D))
    for h in range(H):
        s = q[:, h] @ k[:, h // G].T * scale
        s[np.triu_indices(L, 1)] = -np.inf
        s -= s.max(1, keepdims=True)
        w = np.exp(s)
        w /= w.sum(1, keepdims=True)
        out[:, h] = w @ v[:, h // G]
        mag[:, h] = w @ np.abs(v[:, h // G])
    return out, mag


def run(mk, torch, t, lens, H, KV, D, seed=0, pad=0, tail=0, poison=None, stream=0, spread=1.0):
    """Packed sequences (tail: rows behind the last), rows padded by `pad` heads' worth of other data."""
    dt = tt(torch, t)
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    n = int(off[-1]) + tail
    g = torch.Generator().manual_seed(seed)
    wide = (H + 2 * KV) * D + pad
    buf = torch.randn(max(n, 1), wide, generator=g) * spread
    buf = buf.to(dt).cuda()
    if poison:
        poison(buf, off)
    out = torch.full((max(n, 1), H * D + pad), 7.0, dtype=dt, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    o = torch.as_tensor(off).cuda()
    e = buf.element_size()
    torch.cuda.synchronize()
    mk.attention_prompt(t, buf.data_ptr(), wide, buf.data_ptr() + H * D * e, wide, buf.data_ptr() + (H + KV) * D * e,
                        wide, n, len(lens), o.data_ptr(), H, KV, D, D ** -0.5, out.data_ptr(), H * D + pad,
                        st.data_ptr(), stream)
    torch.cuda.synchronize()
    assert int(st) == 0
    x = buf.float().cpu().numpy().astype(np.float64)
    return x, off, out.float().cpu().numpy(), n


def check(torch, t, x, off, got, H, KV, D, rows=None):
    h = torch.finfo(tt(torch, t)).eps / 2
    tiny = 2.0 ** -25 if t == F16 else 0.0  # half a subnormal step of fp16
    for s in range(len(off) - 1):
        lo, hi = off[s], off[s + 1]
        if lo == hi:
            continue
        q, k, v = (x[lo:hi, a * D:b * D].reshape(hi - lo, -1, D) for a, b in ((0, H), (H, H + KV), (H + KV, H + 2 * KV)))
        want, mag = exact(q, k, v, D ** -0.5)
        y = got[lo:hi, :H * D].reshape(hi - lo, H, D)
        tol = (h + FP32_PART) * mag + h * np.abs(want) + tiny
        bad = ~(np.abs(y - want) <= tol)
        assert not bad.any(), (s, np.argwhere(bad)[:4], np.abs(y - want)[bad][:4], tol[bad][:4])
    assert (got[:, H * D:] == 7).all()
    assert (got[off[-1]:] == 7).all()


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[1], [2], [127], [128], [129], [255], [256], [257], [300, 1, 0, 513, 64], [0, 0, 5, 0]])
def test_lengths(mk, torch_cuda, t, D, lens):
    x, off, got, _ = run(mk, torch_cuda, t, lens, 4, 2, D, seed=len(lens) + lens[0], pad=8, tail=3)
    check(torch_cuda, t, x, off, got, 4, 2, D)


@pytest.mark.parametrize("H,KV", [(1, 1), (8, 8), (8, 1), (6, 2), (5, 1), (40, 8)])
@pytest.mark.parametrize("D", [64, 128])
def test_heads(mk, torch_cuda, H, KV, D):
    x, off, got, _ = run(mk, torch_cuda, BF16, [70, 200], H, KV, D, seed=H)
    check(torch_cuda, BF16, x, off, got, H, KV, D)


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_long(mk, torch_cuda, t, D):
    """Every stage of the ring reused many times, the maximum rising late."""
    def late(buf, off):  # keys that grow along the sequence raise the running maximum again and again
        n = buf.shape[0]
        w = torch_cuda.linspace(0.1, 3.0, n, device="cuda")[:, None]
        buf[:, 2 * D:3 * D] = (buf[:, 2 * D:3 * D].float() * w).to(buf.dtype)
    x, off, got, _ = run(mk, torch_cuda, t, [2500], 2, 1, D, seed=2, poison=late)
    check(torch_cuda, t, x, off, got, 2, 1, D)


def test_many_sequences(mk, torch_cuda):
    """More sequences than a warp has lanes, many of them empty."""
    lens = [(i * 37) % 150 if i % 3 else 0 for i in range(150)]
    x, off, got, _ = run(mk, torch_cuda, BF16, lens, 2, 1, 64, seed=4)
    check(torch_cuda, BF16, x, off, got, 2, 1, 64)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("D", [64, 128])
def test_masked_values_do_not_leak(mk, torch_cuda, value, D):
    """A key and value row that is not finite reaches only the rows that see it: earlier rows, the other sequences and the
    rows behind the last are as if it were not there."""
    torch = torch_cuda
    H, KV, lens, at = 4, 2, [300, 90, 260], 150  # row 150 of each sequence that is that long

    def spoil(buf, off):
        for s in (0, 2):
            buf[off[s] + at, H * D:] = value
        buf[off[1] + 89, (H + KV) * D:] = value  # the last row of the middle one
        buf[off[3]:, :] = value

    x, off, got, n = run(mk, torch, BF16, lens, H, KV, D, seed=8, tail=5, poison=spoil)
    clean = x.copy()
    clean[~np.isfinite(clean)] = 0.0
    for s, first in ((0, at), (1, 89), (2, at)):
        lo, hi = off[s], off[s + 1]
        q, k, v = (clean[lo:hi, a * D:b * D].reshape(hi - lo, -1, D)
                   for a, b in ((0, H), (H, H + KV), (H + KV, H + 2 * KV)))
        want, mag = exact(q[:first], k[:first], v[:first], D ** -0.5)
        y = got[lo:hi, :H * D].reshape(hi - lo, H, D)
        h = 2.0 ** -8
        assert np.all(np.abs(y[:first] - want) <= (h + FP32_PART) * mag + h * np.abs(want)), s
        if s == 1:  # the value alone: the row that sees it takes it
            assert not np.isfinite(y[first:]).any(), s
        elif np.isnan(value):
            assert np.isnan(y[first:]).all(), s
    assert (got[off[-1]:] == 7).all()


def test_finite_values_that_overflow_nothing(mk, torch_cuda):
    """Large scores (weights of 0 and 1) and the type's largest values in V."""
    torch = torch_cuda
    H = KV = 1
    D = 64

    def big(buf, off):
        buf[:, :2 * D] *= 20
        buf[:, 2 * D:] = torch.where(buf[:, 2 * D:] > 0, 60000.0, -60000.0).to(buf.dtype)

    x, off, got, _ = run(mk, torch, F16, [200], H, KV, D, seed=3, poison=big)
    assert np.isfinite(got[:, :D]).all()
    q, k, v = (x[:, a * D:(a + 1) * D].reshape(-1, 1, D) for a in range(3))
    want, mag = exact(q, k, v, D ** -0.5)
    # scores reach 4000: their fp32 error, 2^-17 of it, moves a weight by up to 2^-5 where two of them compete
    assert np.all(np.abs(got[:, :D].reshape(-1, 1, D) - want) <= (2.0 ** -11 + 2.0 ** -4) * mag + 32)


def test_bad_offsets(mk, torch_cuda):
    """Descending offsets, offsets below 0 or past the rows: those sequences are left as they were and recorded."""
    torch = torch_cuda
    H = KV = 1
    D, n = 64, 40
    buf = torch.randn(n, 3 * D, device="cuda").to(torch.bfloat16)
    for off, bad in (([0, 20, 50], 1), ([0, 30, 20], 1), ([-5, 20, 40], 0)):
        o = torch.tensor(off, dtype=torch.int32, device="cuda")
        out = torch.full((n, D), 7.0, dtype=torch.bfloat16, device="cuda")
        st = torch.zeros(1, dtype=torch.int32, device="cuda")
        mk.attention_prompt(BF16, buf.data_ptr(), 3 * D, buf.data_ptr() + 2 * D, 3 * D, buf.data_ptr() + 4 * D, 3 * D, n,
                            2, o.data_ptr(), H, KV, D, 0.125, out.data_ptr(), D, st.data_ptr())
        torch.cuda.synchronize()
        assert int(st) == mk.MK_ERR_ARG
        good = (20, 40) if bad == 0 else (0, off[1])
        rows = np.zeros(n, bool)
        rows[good[0]:good[1]] = True
        y = out.float().cpu().numpy()
        assert (y[~rows] == 7).all() and (y[rows] != 7).any(1).all(), off


def test_host_memory_is_refused(mk, torch_cuda):
    torch = torch_cuda
    x = torch.zeros(4, 3 * 64, dtype=torch.bfloat16)
    d = x.cuda()
    off = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(mk.MalkinError) as e:
        mk.attention_prompt(BF16, d.data_ptr(), 192, x.pin_memory().data_ptr(), 192, d.data_ptr(), 192, 4, 1,
                            off.data_ptr(), 1, 1, 64, 0.125, d.data_ptr(), 192)
    assert e.value.code == mk.MK_ERR_ARG and "dev_k" in str(e.value)


def test_stream_and_graph(mk, torch_cuda):
    """On a stream of its own, two calls at once on two streams, and captured: the replay follows new values and new
    offsets in the same buffers."""
    torch = torch_cuda
    H, KV, D, n = 4, 2, 128, 700
    wide = (H + 2 * KV) * D
    g = torch.Generator().manual_seed(1)
    bufs = [torch.randn(n, wide, generator=g).to(torch.float16).cuda() for _ in range(2)]
    offs = [torch.tensor(o, dtype=torch.int32, device="cuda") for o in ([0, 300, 700], [0, 650, 690])]
    outs = [torch.full((n, H * D), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    call = lambda i, s: mk.attention_prompt(  # noqa: E731
        F16, bufs[i].data_ptr(), wide, bufs[i].data_ptr() + 2 * H * D, wide, bufs[i].data_ptr() + 2 * (H + KV) * D, wide,
        n, 2, offs[i].data_ptr(), H, KV, D, D ** -0.5, outs[i].data_ptr(), H * D, stream=s)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(2):
        call(i, streams[i].cuda_stream)
    torch.cuda.synchronize()

    def verify(i):
        x = bufs[i].float().cpu().numpy().astype(np.float64)
        off = offs[i].cpu().numpy()
        check(torch, F16, x, off, np.pad(outs[i].float().cpu().numpy(), ((0, 0), (0, 1)), constant_values=7), H, KV, D)
    for i in range(2):
        verify(i)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0, torch.cuda.current_stream().cuda_stream)
    bufs[0].copy_(torch.randn(n, wide, generator=g))
    offs[0].copy_(torch.tensor([0, 5, 444]))
    outs[0].fill_(7.0)
    graph.replay()
    torch.cuda.synchronize()
    verify(0)


@pytest.mark.parametrize("n,off,good", [
    (1000, [0, 600, 0, 600, 0, 600, 1000], [0, 5]),  # the same rows three times: the first stands
    (500, [0, 300, 100, 500], [0]),                  # the third begins inside the first
    (500, [100, 300, 0, 400, 450], [0, 3]),          # or reaches over it
    (4, [0, 1, 2, 3, 4] + [4] * 35 + [7], [0, 1, 2, 3]),  # a bad end behind more empty sequences than there are rows
    (40, [0] * 70 + [40, 30], [69])])
def test_offsets_that_are_bad_together(mk, torch_cuda, n, off, good):
    """Every bad offset is recorded, also behind the last row; a sequence over an earlier one's rows is left out, and the
    others are whole."""
    torch = torch_cuda
    H, KV, D = 4, 2, 64
    wide = (H + 2 * KV) * D
    buf = torch.randn(n, wide, generator=torch.Generator().manual_seed(n)).to(torch.bfloat16).cuda()
    o = torch.tensor(off, dtype=torch.int32, device="cuda")
    out = torch.full((n, H * D + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    e = 2
    mk.attention_prompt(BF16, buf.data_ptr(), wide, buf.data_ptr() + H * D * e, wide, buf.data_ptr() + (H + KV) * D * e,
                        wide, n, len(off) - 1, o.data_ptr(), H, KV, D, D ** -0.5, out.data_ptr(), H * D + 8, st.data_ptr())
    torch.cuda.synchronize()
    assert int(st) == mk.MK_ERR_ARG
    x, got = buf.float().cpu().numpy().astype(np.float64), out.float().cpu().numpy()
    rest = np.ones(n, bool)
    for s in good:
        lo, hi = off[s], off[s + 1]
        check(torch, BF16, x[lo:hi], [0, hi - lo], got[lo:hi], H, KV, D)
        rest[lo:hi] = False
    assert (got[rest] == 7).all()


def test_many_small_weights(mk, torch_cuda):
    """One key of weight 1 with a value of 0 and 1999 of weight 2^-25.4: together they are the output. fp16 holds weights
    below its smallest normal number to 2^-32 of the largest (it keeps them 2^7 larger), so the row's sum is off by at most
    half of that for each, on top of the rounding of the output."""
    torch = torch_cuda
    H = KV = 1
    D, n, shift = 64, 2000, -17.609375

    def one(buf, off):
        buf[:] = 0
        buf[:, 0] = 8.0           # the score of a key is its first value
        buf[1:, D] = shift
        buf[1:, 2 * D:] = 1.0

    x, off, got, _ = run(mk, torch, F16, [n], H, KV, D, poison=one)
    w = np.exp(shift)
    i = np.arange(n)
    want = i * w / (1 + i * w)
    tol = i * 2.0 ** -32 + (2.0 ** -11 + 2.0 ** -12) * want + 2.0 ** -25
    err = np.abs(got[:, :D] - want[:, None])
    assert np.all(err <= tol[:, None]), (err.max(), want[-1], got[-1, 0])
