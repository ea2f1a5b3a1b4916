"""mk_attention_shared on the GPU against softmax attention in 64 bits over each token's own list of keys."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F16, BF16 = 1, 30

# Error of an output beside A = sum_j w_j |v_j|: weights x scales are rounded to fp16 (2^-11 of each); fp32 parts (scores of
# D products, exponents, sums, joining) together below 2^-11 A for scores below 24, as in the prompt attention's test;
# then half a step of the output's type.
W_PART = 2.0 ** -11 + 2.0 ** -11


def tt(torch, t):
    return {F16: torch.float16, BF16: torch.bfloat16}[t]


class Batch:
    """Requests behind prefixes: groups = [(prefix_len, [request, ...])], request = (own contiguous keys before the first
    token, tokens) or (own keys, "tree", depth)."""

    def __init__(self, rng, groups, KV, D, loose=0, spare=5):
        self.group_off, self.prefix_base, self.prefix_len = [0], [], []
        self.kv_base, self.n_keys, self.anc = [], [], []
        at = spare
        for P, reqs in groups:
            self.prefix_base.append(at)
            self.prefix_len.append(P)
            at += P + spare
            for r in reqs:
                at = self.request(r, at) + spare
            self.group_off.append(len(self.kv_base))
        for _ in range(loose):  # tokens of no group
            at = self.request((7, 1), at) + spare
        self.rows = at
        self.n = len(self.kv_base)
        self.k = rng.integers(-127, 128, (KV, at, D)).astype(np.int8)
        self.v = rng.integers(-127, 128, (KV, at, D)).astype(np.int8)
        self.ks = rng.uniform(0.002, 0.02, (KV, at)).astype(np.float32)
        self.vs = rng.uniform(0.002, 0.02, (KV, at)).astype(np.float32)

    def request(self, r, at):
        if r[1] == "tree":
            keys, _, depth = r
            paths = [[]]
            self.add(at, keys, [])
            for i in range(depth):
                up = paths[0 if i == 0 else 2 * i - 1]
                for c in (1, 2):
                    p = up + [keys + 2 * i + c - 1]
                    paths.append(p)
                    self.add(at, keys, p)
            return at + keys + 2 * depth
        keys, toks = r
        for i in range(toks):
            self.add(at, keys + i, [])
        return at + keys + toks

    def add(self, base, keys, anc):
        self.kv_base.append(base)
        self.n_keys.append(keys)
        self.anc.append(anc)

    def keys_of(self, t):
        rows = []
        for g in range(len(self.prefix_len)):
            if self.group_off[g] <= t < self.group_off[g + 1]:
                rows += list(range(self.prefix_base[g], self.prefix_base[g] + self.prefix_len[g]))
        rows += list(range(self.kv_base[t], self.kv_base[t] + self.n_keys[t]))
        return rows + [self.kv_base[t] + a for a in self.anc[t]]


def call(mk, torch, t, b, q, H, KV, D, stream=0, keep=None, status=0):
    off = np.concatenate([[0], np.cumsum([len(a) for a in b.anc])])
    flat = [x for a in b.anc for x in a]
    arrays = [b.k, b.v, b.ks, b.vs, b.group_off, b.prefix_base or [0], b.prefix_len or [0], b.kv_base, b.n_keys, off,
              flat or [0]]
    d = [torch.as_tensor(np.asarray(a) if i < 4 else np.asarray(a, np.int32)).cuda() for i, a in enumerate(arrays)]
    out = torch.full((b.n, q.shape[1]), 7.0, dtype=q.dtype, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = torch.empty(mk.attention_shared_workspace(b.n, H, KV, D, len(b.prefix_len)), dtype=torch.uint8, device="cuda")
    ws.fill_(255)  # whatever an earlier user left there (NaN as floats)
    torch.cuda.synchronize()
    go = lambda s: mk.attention_shared(  # noqa: E731
        t, q.data_ptr(), q.shape[1], b.n, H, KV, D, D ** -0.5, d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(),
        d[3].data_ptr(), b.k.shape[1], len(b.prefix_len), d[4].data_ptr(), d[5].data_ptr(), d[6].data_ptr(),
        d[7].data_ptr(), d[8].data_ptr(), d[9].data_ptr(), d[10].data_ptr(), len(flat), out.data_ptr(), q.shape[1],
        ws.data_ptr(), ws.numel(), st.data_ptr(), s)
    if keep is not None:
        keep.update(go=go, d=d, out=out, st=st, ws=ws)
    go(stream)
    torch.cuda.synchronize()
    assert int(st) == status
    return out.float().cpu().numpy()


def check(torch, t, b, q, got, H, KV, D, tokens=None):
    h = torch.finfo(tt(torch, t)).eps / 2
    x = q.float().cpu().numpy().astype(np.float64)
    G = H // KV
    k = b.k.astype(np.float64) * b.ks[..., None].astype(np.float64)
    v = b.v.astype(np.float64) * b.vs[..., None].astype(np.float64)
    for i in range(b.n) if tokens is None else tokens:
        rows = b.keys_of(i)
        if not rows:
            assert (got[i, :H * D] == 0).all(), i
            continue
        for kv in range(KV):
            s = x[i, kv * G * D:(kv + 1) * G * D].reshape(G, D) @ k[kv, rows].T * D ** -0.5
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            want, mag = w @ v[kv, rows], w @ np.abs(v[kv, rows])
            y = got[i, kv * G * D:(kv + 1) * G * D].reshape(G, D)
            tol = W_PART * mag + h * np.abs(want) + (2.0 ** -25 if t == F16 else 0.0)
            bad = ~(np.abs(y - want) <= tol)
            assert not bad.any(), (i, kv, np.argwhere(bad)[:3], np.abs(y - want)[bad][:3], tol[bad][:3])
    assert (got[:, H * D:] == 7).all()


def queries(torch, t, n, H, D, seed=0, pad=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, H * D + pad, generator=g).to(tt(torch, t)).cuda()


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("groups,loose", [
    ([(1, [(0, 1)])], 0),                                             # one token, one key
    ([(0, [(0, 1)])], 0),                                             # no key at all: zeros
    ([(64, [(0, 1), (1, 1)])], 0), ([(65, [(63, 2), (64, 3)])], 0),   # around the block of 64 keys
    ([(200, [(5, 1)] * 3), (0, [(9, 2)]), (130, [(0, 4), (300, 1)])], 2),
    ([(500, [(40, "tree", 4), (77, "tree", 1), (0, "tree", 2)])], 1),
    ([], 3),                                                          # no prefix anywhere
    ([(1500, [(20 * i, 3) for i in range(20)])], 0)])                 # more rows than a tile
def test_batches(mk, torch_cuda, t, D, groups, loose):
    H, KV = 8, 2
    b = Batch(np.random.default_rng(D + len(groups)), groups, KV, D, loose)
    q = queries(torch_cuda, t, b.n, H, D, 1, pad=8)
    check(torch_cuda, t, b, q, call(mk, torch_cuda, t, b, q, H, KV, D), H, KV, D)


@pytest.mark.parametrize("H,KV", [(1, 1), (8, 8), (5, 1), (40, 8), (6, 2), (128, 1), (130, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_heads(mk, torch_cuda, H, KV, D):
    b = Batch(np.random.default_rng(H), [(150, [(30, 2), (3, "tree", 2)]), (70, [(0, 1)])], KV, D, 1)
    q = queries(torch_cuda, BF16, b.n, H, D, H)
    check(torch_cuda, BF16, b, q, call(mk, torch_cuda, BF16, b, q, H, KV, D), H, KV, D)


@pytest.mark.parametrize("t", [F16, BF16])
def test_long_prefix_and_many_requests(mk, torch_cuda, t):
    """Pieces that span several units, units cut into many pieces, more tokens than the plan's block has threads."""
    H, KV, D = 4, 2, 128
    rng = np.random.default_rng(5)
    b = Batch(rng, [(9000, [(int(rng.integers(0, 40)), 1) for _ in range(700)]),
                    (333, [(int(rng.integers(0, 200)), 2) for _ in range(300)])], KV, D)
    q = queries(torch_cuda, t, b.n, H, D, 9)
    got = call(mk, torch_cuda, t, b, q, H, KV, D)
    check(torch_cuda, t, b, q, got, H, KV, D, tokens=list(range(0, b.n, 37)) + [699, 700, b.n - 1])


def test_rising_maximum(mk, torch_cuda):
    """Scores that grow along the prefix raise the running maximum in every block; one huge key at the end."""
    torch = torch_cuda
    H, KV, D = 4, 1, 128
    b = Batch(np.random.default_rng(1), [(2000, [(10, 2)])], KV, D)
    lo = b.prefix_base[0]
    b.ks[0, lo:lo + 2000] = np.linspace(1e-4, 0.05, 2000)
    b.k[0, lo + 1999] = 127
    q = (queries(torch, BF16, b.n, H, D, 2).float().abs() * 0.1).to(torch.bfloat16)
    check(torch, BF16, b, q, call(mk, torch, BF16, b, q, H, KV, D), H, KV, D)


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("H,KV,D", [(8, 2, 128), (16, 8, 64), (5, 1, 128)])
def test_pieces_of_every_length(mk, torch_cuda, t, H, KV, D):
    """Batches whose parts are one block or many, alone and dual, so that pieces end at every place in a unit."""
    torch = torch_cuda
    for seed in range(4):
        rng = np.random.default_rng(seed)
        groups = []
        for _ in range(int(rng.integers(1, 6))):
            reqs = [(int(rng.integers(0, 400)), int(rng.integers(1, 5))) for _ in range(int(rng.integers(1, 24)))]
            groups.append((int(rng.integers(0, 1500)) if rng.random() < 0.7 else int(rng.integers(0, 97)), reqs))
        b = Batch(rng, groups, KV, D, loose=seed)
        q = queries(torch, t, b.n, H, D, seed)
        check(torch, t, b, q, call(mk, torch, t, b, q, H, KV, D), H, KV, D)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_rows_outside_the_tables(mk, torch_cuda, value):
    """Scales of rows that no token looks at, and of rows that only later tokens of the request look at, may hold
    anything."""
    torch = torch_cuda
    H, KV, D = 4, 2, 64
    b = Batch(np.random.default_rng(3), [(100, [(20, 3), (5, "tree", 2)])], KV, D, 1)
    q = queries(torch, F16, b.n, H, D, 4)
    seen = set(r for t in range(b.n) for r in b.keys_of(t))
    for r in range(b.rows):
        if r not in seen:
            b.ks[:, r] = b.vs[:, r] = value
    check(torch, F16, b, q, call(mk, torch, F16, b, q, H, KV, D), H, KV, D)
    last = b.kv_base[0] + 21  # the row only the third token of the first request sees
    b.ks[:, last] = b.vs[:, last] = value
    got = call(mk, torch, F16, b, q, H, KV, D)
    check(torch, F16, b, q, got, H, KV, D, tokens=[t for t in range(b.n) if t != 2])
    assert not np.isfinite(got[2, :H * D]).any()


def test_zero_scale_and_extreme_values(mk, torch_cuda):
    """Rows of zeros (scale 0) and the int8 range's ends."""
    torch = torch_cuda
    H, KV, D = 8, 2, 128
    b = Batch(np.random.default_rng(8), [(90, [(3, 2)])], KV, D)
    b.k[:, ::3], b.v[:, ::5] = 127, -128
    b.k[:, 1::7] = -128
    b.ks[:, ::11] = 0
    b.vs[:, ::13] = 0
    for t in (F16, BF16):
        q = queries(torch, t, b.n, H, D, 6)
        check(torch, t, b, q, call(mk, torch, t, b, q, H, KV, D), H, KV, D)


def test_bad_tables(mk, torch_cuda):
    """Tables that leave the cache or the batch: recorded; the tokens they do not concern keep their results."""
    torch = torch_cuda
    H, KV, D = 4, 2, 64
    make = lambda: Batch(np.random.default_rng(2), [(80, [(10, 2)]), (40, [(6, "tree", 2)])], KV, D, 1)  # noqa: E731
    good = make()
    q = queries(torch, BF16, good.n, H, D, 3)
    base = call(mk, torch, BF16, good, q, H, KV, D)
    check(torch, BF16, good, q, base, H, KV, D)
    first, second, last = [0, 1], list(range(2, 7)), [7]

    def spoiled(change, hurt):
        b = make()
        change(b)
        got = call(mk, torch, BF16, b, q, H, KV, D, status=mk.MK_ERR_ARG)
        for t in range(b.n):
            if t not in hurt:
                assert np.array_equal(got[t], base[t]), t
        return got

    def group_base(b): b.prefix_base[0] = b.rows - 10
    def group_neg(b): b.prefix_len[0] = -1
    def group_tokens(b): b.group_off[2] = b.n + 5
    def token_keys(b): b.n_keys[1] = b.rows
    def token_base(b): b.kv_base[7] = -3
    def ancestor(b): b.anc[6][-1] = b.rows
    spoiled(group_base, first)
    spoiled(group_neg, first)
    spoiled(group_tokens, second)
    spoiled(token_keys, [1])
    spoiled(token_base, last)
    spoiled(ancestor, [6])
    b = make()  # groups over one another: only that nothing outside the buffers is touched
    b.group_off = [0, 7, 0, 7, 0, 7]
    b.prefix_base, b.prefix_len = [5] * 5, [30] * 5
    call(mk, torch, BF16, b, q, H, KV, D, status=mk.MK_ERR_ARG)
    b.group_off = [0, 7] * 1300
    b.prefix_base, b.prefix_len = [5] * 2599, [30] * 2599
    call(mk, torch, BF16, b, q, H, KV, D, status=mk.MK_ERR_ARG)


def test_streams_and_graph(mk, torch_cuda):
    """Two calls at once on two streams with a workspace each; captured, and replayed with other tables and values."""
    torch = torch_cuda
    H, KV, D = 8, 2, 128
    rng = np.random.default_rng(4)
    bs = [Batch(rng, [(600, [(20, 2), (7, "tree", 3)])], KV, D), Batch(rng, [(900, [(3, 4)] * 6)], KV, D)]
    qs = [queries(torch, F16, b.n, H, D, i) for i, b in enumerate(bs)]
    keep = [{}, {}]
    for i in range(2):
        call(mk, torch, F16, bs[i], qs[i], H, KV, D, keep=keep[i])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for i in range(2):
            keep[i]["out"].fill_(7.0)
        torch.cuda.synchronize()
        for i in range(2):
            keep[i]["go"](streams[i].cuda_stream)
        torch.cuda.synchronize()
        for i in range(2):
            check(torch, F16, bs[i], qs[i], keep[i]["out"].float().cpu().numpy(), H, KV, D)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep[0]["go"](torch.cuda.current_stream().cuda_stream)
    b = bs[0]
    b.prefix_len[0] = 333
    b.n_keys[1] -= 4
    keep[0]["d"][6].copy_(torch.tensor(b.prefix_len, dtype=torch.int32))
    keep[0]["d"][8].copy_(torch.tensor(b.n_keys, dtype=torch.int32))
    qs[0].copy_(torch.randn(qs[0].shape))
    graph.replay()
    torch.cuda.synchronize()
    check(torch, F16, b, qs[0], keep[0]["out"].float().cpu().numpy(), H, KV, D)


def test_agrees_with_the_exact_attention(mk, torch_cuda):
    """Beside mk_attention: the same cache and tables with every request's prefix as its own rows."""
    torch = torch_cuda
    H, KV, D = 8, 2, 128
    b = Batch(np.random.default_rng(6), [(0, [(150, 3), (90, "tree", 3)])], KV, D)
    q = queries(torch, F16, b.n, H, D, 5)
    keep = {}
    got = call(mk, torch, F16, b, q, H, KV, D, keep=keep)
    d = keep["d"]
    out = torch.zeros(b.n, H * D, device="cuda")
    q32 = q.float()
    mk.attention(q32.data_ptr(), b.n, H, KV, D, d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), d[3].data_ptr(), b.rows,
                 d[7].data_ptr(), d[8].data_ptr(), d[9].data_ptr(), d[10].data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    want = out.cpu().numpy()
    # both within their own error of the exact value; |v| <= 2.6 here
    assert np.abs(got - want).max() <= (W_PART + 2.0 ** -11) * 2.6


@pytest.mark.parametrize("value", [1e30, 1e12, -1e30])
@pytest.mark.parametrize("t", [F16, BF16])
def test_v_scales_of_keys_a_row_does_not_see(mk, torch_cuda, t, value):
    """A row of the cache that only later tokens of the request look at may have any finite scale."""
    H, KV, D = 4, 2, 64
    b = Batch(np.random.default_rng(3), [(100, [(20, 3), (5, "tree", 2)])], KV, D, 1)
    q = queries(torch_cuda, t, b.n, H, D, 4)
    b.vs[:, b.kv_base[0] + 21] = value  # the row that only the third token of the first request sees
    got = call(mk, torch_cuda, t, b, q, H, KV, D)
    check(torch_cuda, t, b, q, got, H, KV, D, tokens=[i for i in range(b.n) if i != 2])


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_v_scales_far_apart(mk, torch_cuda, t, D):
    """Scales of V over many powers of two, the largest of them on keys of hardly any weight: no product that counts is
    lost. (A product weight x scale is rounded by 2^-11 of itself or by 2^-31 of the row's largest in the block; with |v|
    between 32 and 127 and 700 keys the latter stay below 700 x 4 x 2^-31 of sum w |v|.)"""
    H, KV = 8, 2
    for seed in range(3):
        rng = np.random.default_rng(seed)
        b = Batch(rng, [(500, [(40, 2), (90, "tree", 2), (200, 1)]), (0, [(97, 2)])], KV, D, 1)
        b.v = (rng.integers(32, 128, b.v.shape) * rng.choice([-1, 1], b.v.shape)).astype(np.int8)
        b.vs = (10.0 ** rng.uniform(-5, 2, b.vs.shape)).astype(np.float32)
        q = queries(torch_cuda, t, b.n, H, D, seed)
        # keys that every query is far from: scores some 40 below the others, V scales of 10^9
        q[:, ::D] = 8.0
        b.k[:, :, 0] = 0
        far = rng.random(b.rows) < 0.03
        b.k[:, far, 0] = -127
        b.ks[:, far] = 40.0 * D ** 0.5 / (8 * 127)
        b.k[:, far, 1:] = 0
        b.vs[:, far] = 1e9
        check(torch_cuda, t, b, q, call(mk, torch_cuda, t, b, q, H, KV, D), H, KV, D)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_ancestor_with_a_scale_that_is_not_finite(mk, torch_cuda, value):
    """A V scale that is not finite makes the tokens NaN that have its row for an ancestor, as those that have it among
    their own keys, and nobody else."""
    torch = torch_cuda
    H, KV, D = 4, 2, 64
    b = Batch(np.random.default_rng(3), [(100, [(20, 3), (5, "tree", 3)])], KV, D, 1)
    q = queries(torch, BF16, b.n, H, D, 4)
    first = 3  # the tree's root token; its next two rows are its children
    row = b.kv_base[first] + 5
    b.vs[:, row] = value
    hit = [i for i in range(b.n) if row in b.keys_of(i)]
    assert 1 < len(hit) < b.n - 4
    got = call(mk, torch, BF16, b, q, H, KV, D)
    check(torch, BF16, b, q, got, H, KV, D, tokens=[i for i in range(b.n) if i not in hit])
    assert np.isnan(got[hit, :H * D]).all()


@pytest.mark.parametrize("off", [[0, 4, 0, 7], [0, 4, 2, 6, 7], [0, 4, 4, 1, 4, 0, 7], [0, 4] + [0, 7] * 600])
def test_groups_over_one_another(mk, torch_cuda, off):
    """A group with tokens of an earlier one has none of its keys; the earlier one keeps its own, and every token its own
    rows."""
    torch = torch_cuda
    H, KV, D = 4, 2, 64
    b = Batch(np.random.default_rng(2), [(80, [(10, 2), (3, 2)]), (0, [(6, 1), (4, 2)])], KV, D, 1)
    assert b.n == 8
    q = queries(torch, BF16, b.n, H, D, 3)
    base = b.prefix_base[0]
    G = len(off) - 1
    good = [off[g] < off[g + 1] and off[g] >= max([off[e + 1] for e in range(g) if off[e] < off[e + 1]] + [0])
            for g in range(G)]
    plain = b.keys_of
    b.prefix_base, b.prefix_len = [base + g % 7 for g in range(G)], [80 - g % 11 - g % 7 for g in range(G)]
    if G > 1000:
        b.prefix_base, b.prefix_len = [base] * G, [80] + [30] * (G - 1)
    b.group_off = off

    def keys_of(i):
        rows = []
        for g in range(G):
            if good[g] and off[g] <= i < off[g + 1]:
                rows += list(range(b.prefix_base[g], b.prefix_base[g] + b.prefix_len[g]))
        rows += list(range(b.kv_base[i], b.kv_base[i] + b.n_keys[i]))
        return rows + [b.kv_base[i] + a for a in b.anc[i]]
    b.keys_of = keys_of
    got = call(mk, torch, BF16, b, q, H, KV, D, status=mk.MK_ERR_ARG)
    check(torch, BF16, b, q, got, H, KV, D)


@pytest.mark.parametrize("H,KV", [(8, 2), (6, 2)])  # 32 and 42 tokens a stream (126 of its 128 rows)
@pytest.mark.parametrize("keys", [95, 96, 97, 191, 192, 193])
def test_around_blocks_and_tiles(mk, torch_cuda, H, KV, keys):
    """Prefixes and own rows that end at a block of 96 keys, one before and one behind it; groups and runs of as many tokens
    as a stream or a tile of two streams takes, one fewer and one more."""
    torch = torch_cuda
    D, half = 64, 128 // (H // KV)
    groups = [(keys, [(keys - 1, 1), (keys, 2)])]
    groups += [(keys if toks % 2 else 0, [(keys - 2, toks)]) for toks in (half - 1, half, half + 1)]
    groups += [(keys, [(3, 1)] * toks) for toks in (2 * half - 1, 2 * half, 2 * half + 1)]
    b = Batch(np.random.default_rng(keys), groups, KV, D, 1)
    for t in (F16, BF16):
        q = queries(torch, t, b.n, H, D, keys)
        check(torch, t, b, q, call(mk, torch, t, b, q, H, KV, D), H, KV, D)


@pytest.mark.parametrize("cached", [1, 300])
def test_prompt_rows_behind_cached_ones(mk, torch_cuda, cached):
    """The rest of a prompt whose first rows are in the cache: a run of tokens over one sequence whose n_keys rise by one,
    more of them than a tile takes."""
    torch = torch_cuda
    H, KV, D = 8, 2, 128
    b = Batch(np.random.default_rng(cached), [(0, [(cached, 200)]), (64, [(cached + 1, 70)])], KV, D)
    for i in range(b.n):
        b.n_keys[i] += 1  # each token sees its own row, which is in the cache before the call
    q = queries(torch, BF16, b.n, H, D, 1)
    check(torch, BF16, b, q, call(mk, torch, BF16, b, q, H, KV, D), H, KV, D)
