"""Cases of the 16-bit serving operators: q/k norm with rotation, attention over packed prompts, attention over a shared
prefix, and whole-vocabulary verification of drafted tokens. `run` computes each in plain torch operations, or, with
`own` true, through the library's entry points; `exact` restates each from its definition in 64 bits.

The head counts, head width, vocabulary and tree sizes are those of the repository's benchmark configurations: 16 / 32 /
40 query heads over 8 KV heads of 128 values, 151936 tokens, trees of 17 rows, prefixes of 512 to 8192 tokens."""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IDS = {"f32": 0, "f16": 1, "bf16": 30}
EPS = 1e-6


def listed():
    return [
        # one tree of 17 rows at decode time, float activations: latency
        {"name": "norm_rope_tree_f32", "op": "norm_rope", "type": "f32", "n": 17, "H": 32, "KV": 8, "D": 128,
         "cache": False, "pad": 0},
        # a prompt chunk of an odd length with narrow heads, rows padded to a wider pitch
        {"name": "norm_rope_chunk_f16", "op": "norm_rope", "type": "f16", "n": 1003, "H": 24, "KV": 8, "D": 64,
         "cache": False, "pad": 8},
        # a whole prefill batch, q and k for the prompt attention and the int8 cache rows in the same pass
        {"name": "norm_rope_prefill_bf16", "op": "norm_rope", "type": "bf16", "n": 16384, "H": 32, "KV": 8, "D": 128,
         "cache": True, "pad": 0},
        # one short prompt: latency
        {"name": "prompt_short_bf16", "op": "prompt", "type": "bf16", "n_seq": 1, "longest": 100, "ragged": False,
         "H": 16, "KV": 8, "D": 128, "mix": 0},
        # eight requests of different lengths packed into one batch
        {"name": "prompt_packed_bf16", "op": "prompt", "type": "bf16", "n_seq": 8, "longest": 2048, "ragged": True,
         "H": 32, "KV": 8, "D": 128, "mix": 1},
        # one long prompt
        {"name": "prompt_long_f16", "op": "prompt", "type": "f16", "n_seq": 1, "longest": 8192, "ragged": False,
         "H": 40, "KV": 8, "D": 128, "mix": 0},
        # four requests with one token each behind a common system prompt: latency
        {"name": "shared_small_bf16", "op": "shared", "type": "bf16", "n_groups": 1, "reqs": 4, "toks": 1,
         "prefix": 1000, "own_keys": 60, "tree": False, "H": 16, "KV": 8, "D": 128, "mix": 2},
        # eight requests, each with a tree of 17 rows, behind one prefix
        {"name": "shared_trees_f16", "op": "shared", "type": "f16", "n_groups": 1, "reqs": 8, "toks": 17,
         "prefix": 2048, "own_keys": 300, "tree": True, "H": 32, "KV": 8, "D": 128, "mix": 2},
        # two prefixes of different lengths with 32 requests each, four chain rows a request
        {"name": "shared_large_bf16", "op": "shared", "type": "bf16", "n_groups": 2, "reqs": 32, "toks": 4,
         "prefix": 32768, "own_keys": 1024, "tree": False, "H": 32, "KV": 8, "D": 128, "mix": 2},
        # one request with eight drafts: latency
        {"name": "verify_one_f32", "op": "verify", "type": "f32", "reqs": 1, "drafts": 8, "ragged": False, "V": 151936,
         "probs": True, "mix": 0},
        # eight requests of up to eight drafts without draft probabilities (drafts taken from the text itself)
        {"name": "verify_lookup_bf16", "op": "verify", "type": "bf16", "reqs": 8, "drafts": 8, "ragged": True,
         "V": 151936, "probs": False, "mix": 1},
        # a large batch
        {"name": "verify_batch_f32", "op": "verify", "type": "f32", "reqs": 64, "drafts": 4, "ragged": False,
         "V": 151936, "probs": True, "mix": 0},
    ]


def _span(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "prompt", "shared", "verify"])
    kv = rng.choice([1, 2, 4, 8])
    c = {"op": op}
    if op == "verify":
        reqs = _span(rng, 1, 64)
        c.update(type=rng.choice(["f32", "f16", "bf16"]), reqs=reqs, drafts=rng.randint(0, 8 if reqs <= 32 else 4),
                 ragged=rng.random() < 0.5, V=rng.choice([151936, _span(rng, 1000, 151936)]), probs=rng.random() < 0.6,
                 mix=rng.randrange(1000))
        return c
    c.update(type=rng.choice(["f16", "bf16"]), H=kv * rng.choice([1, 2, 3, 4, 5, 8]), KV=kv, D=rng.choice([64, 128]))
    if op == "norm_rope":
        c.update(type=rng.choice(["f32", "f16", "bf16"]), n=_span(rng, 1, 8192), cache=rng.random() < 0.3,
                 pad=8 * rng.randint(0, 3))
    elif op == "prompt":
        longest = _span(rng, 1, 4096)
        c.update(longest=longest, n_seq=_span(rng, 1, max(1, min(16, 16384 // longest))), ragged=rng.random() < 0.7,
                 mix=rng.randrange(1000))
    else:
        groups, reqs, tree = rng.randint(1, 3), _span(rng, 1, 16), rng.random() < 0.4
        toks = 2 * rng.randint(1, 8) + 1 if tree else rng.randint(1, 5)
        c.update(n_groups=groups, reqs=reqs, toks=toks, prefix=_span(rng, 16, 16384), own_keys=_span(rng, 1, 1024),
                 tree=tree, mix=rng.randrange(1000))
    return c


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _lengths(case):
    """Lengths of a batch's parts, the first the longest: they go by the case, the values by the seed."""
    mix = random.Random(case["mix"])
    if case["op"] == "prompt":
        L = case["longest"]
        return [L] + [mix.randint(1, L) if case["ragged"] else L for _ in range(case["n_seq"] - 1)]
    if case["op"] == "verify":
        k = case["drafts"]
        return [k] + [mix.randint(0, k) if case["ragged"] else k for _ in range(case["reqs"] - 1)]
    P, own_keys = case["prefix"], case["own_keys"]
    prefix = [P] + [mix.randint(max(1, P // 2), P) for _ in range(case["n_groups"] - 1)]
    return prefix, [own_keys] + [mix.randint(0, own_keys) for _ in range(case["n_groups"] * case["reqs"] - 1)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    dt = DTYPES[case["type"]]
    s["dt"] = dt
    if case["op"] == "norm_rope":
        n, H, KV, D = case["n"], case["H"], case["KV"], case["D"]
        ld = (H + 2 * KV) * D + case["pad"]
        s["ld"] = ld
        s["qkv"] = (_randn(gen, n, ld) * 1.5).to(dt)
        s["q_norm"] = 1 + 0.2 * _randn(gen, D)
        s["k_norm"] = 1 + 0.2 * _randn(gen, D)
        s["n_pos"] = 40960
        ang = torch.arange(s["n_pos"], device="cuda", dtype=torch.float64)[:, None] * torch.pow(
            torch.tensor(1e6, dtype=torch.float64, device="cuda"),
            -torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2))[None, :]
        s["rope"] = torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()
        first = int(torch.randint(0, s["n_pos"] - n + 1, (1,), generator=gen, device="cuda"))
        s["pos"] = torch.arange(first, first + n, device="cuda", dtype=torch.int32)
        s["q_out"] = torch.zeros(n, H, D, dtype=dt, device="cuda")
        s["k_out"] = torch.zeros(n, KV, D, dtype=dt, device="cuda")
        if case["cache"]:
            # the cache of one layer, its rows in an order of their own
            s["kv_at"] = torch.randperm(n, generator=gen, device="cuda").to(torch.int32)
            s["k8"], s["v8"] = (torch.zeros(KV, n, D, dtype=torch.int8, device="cuda") for _ in range(2))
            s["ks"], s["vs"] = (torch.zeros(KV, n, dtype=torch.float32, device="cuda") for _ in range(2))
            s["k_held"], s["v_held"] = (torch.zeros(KV, n, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    elif case["op"] == "prompt":
        H, KV, D, longest = case["H"], case["KV"], case["D"], case["longest"]
        lens = _lengths(case)
        off = [0]
        for x in lens:
            off.append(off[-1] + x)
        n = off[-1]
        s.update(n=n, off=_ints(off), lens=lens)
        at = torch.arange(longest, device="cuda")[None, :]
        held = at < torch.tensor(lens, device="cuda")[:, None]
        s["row"] = torch.where(held, s["off"][:-1, None].long() + at, 0)  # the plain form's padded rows
        s["held"] = held
        # q and k as they leave their norm, v where the projection left it
        s["q"] = _randn(gen, n, H, D).to(dt)
        s["k"] = _randn(gen, n, KV, D).to(dt)
        s["v"] = _randn(gen, n, KV, D).to(dt)
        s["out"] = torch.zeros(n, H, D, dtype=dt, device="cuda")
    elif case["op"] == "shared":
        H, KV, D, T = case["H"], case["KV"], case["D"], case["toks"]
        groups, R = case["n_groups"], case["n_groups"] * case["reqs"]
        n = R * T
        prefix, owned = _lengths(case)
        base, at = [], 0
        for x in prefix:
            base.append(at)
            at += x
        kv_base, n_keys, anc_off, anc = [], [], [0], []
        for x in owned:
            path = {0: []}
            for t in range(T):
                kv_base.append(at)
                if case["tree"]:  # root, then a chain with one sibling a depth; the root's row ends the contiguous keys
                    n_keys.append(x + 1)
                    if t:
                        parent = 0 if t <= 2 else 2 * ((t - 1) // 2) - 1
                        path[t] = path[parent] + [x + t]
                    anc += path[t]
                else:
                    n_keys.append(x + t + 1)
                anc_off.append(len(anc))
            at += x + T
        s.update(n=n, n_rows=at, group_off=_ints([g * case["reqs"] * T for g in range(groups + 1)]),
                 prefix_base=_ints(base), prefix_len=_ints(prefix), kv_base=_ints(kv_base), n_keys=_ints(n_keys),
                 anc_off=_ints(anc_off), anc=_ints(anc or [0]))
        for name in ("k", "v"):
            x = _randn(gen, KV, at, D) * (1.0 if name == "k" else 0.5)
            scale = x.abs().amax(-1) / 127
            s[name + "s"] = scale
            s[name + "8"] = torch.round(x / scale[..., None]).to(torch.int8)
        s["q"] = _randn(gen, n, H, D).to(dt)
        s["out"] = torch.zeros(n, H, D, dtype=dt, device="cuda")
        # the plain form's padded tables: rows of every key a token attends to besides its prefix
        wide = max(n_keys)
        deep = max(b - a for a, b in zip(anc_off, anc_off[1:]))
        rows, kept = torch.zeros(n, deep, dtype=torch.int64), torch.zeros(n, deep, dtype=torch.bool)
        for t in range(n if deep else 0):
            m = anc_off[t + 1] - anc_off[t]
            rows[t, :m] = torch.tensor(anc[anc_off[t]:anc_off[t + 1]], dtype=torch.int64) + kv_base[t]
            kept[t, :m] = True
        s["anc_row"], s["anc_kept"] = rows.cuda(), kept.cuda()
        first = s["kv_base"].view(R, T)[:, :1].long()
        s["own_row"] = (first + torch.arange(wide, device="cuda")).clamp(max=at - 1)
        s["own_kept"] = torch.arange(wide, device="cuda") < s["n_keys"].view(R, T, 1)
        span = torch.arange(max(prefix), device="cuda")
        s["pre_row"] = (s["prefix_base"].long()[:, None] + span).clamp(max=at - 1)
        s["pre_kept"] = span < s["prefix_len"][:, None]
    else:
        R, V = case["reqs"], case["V"]
        kk = _lengths(case)
        off = [0]
        for x in kk:
            off.append(off[-1] + x + 1)
        m, nd = off[-1], off[-1] - R
        s.update(m=m, nd=nd, row_off=_ints(off))
        logits = _randn(gen, m, V) * 2.5
        # temperatures as users set them, some requests greedy
        temp = torch.tensor([0.0 if R > 3 and r % 4 == 3 else 0.6 + 0.1 * (r % 7) for r in range(R)])
        s["temp"] = temp.float().cuda()
        of = torch.repeat_interleave(torch.arange(R), torch.tensor(kk) + 1).cuda()
        is_last = torch.zeros(m, dtype=torch.bool, device="cuda")
        is_last[s["row_off"][1:].long() - 1] = True
        s["draft_row"] = torch.nonzero(~is_last).flatten()
        s["row_req"] = of
        T = torch.where(s["temp"] > 0, s["temp"], 1.0)[of[s["draft_row"]]]
        if nd:
            # a draft model that is near the target; greedy requests draft its best token
            near = (logits[s["draft_row"]] + 0.6 * _randn(gen, nd, V)) / T[:, None]
            q = torch.softmax(near, -1)
            drawn = torch.multinomial(q, 1, generator=gen).flatten()
            greedy = s["temp"][of[s["draft_row"]]] <= 0
            s["draft"] = torch.where(greedy, near.argmax(-1), drawn).to(torch.int32)
        else:
            q = torch.zeros(1, V, device="cuda")
            s["draft"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        if case["probs"]:
            s["q"] = q
        s["logits"] = logits.to(dt)
        s["u"] = torch.rand(m, generator=gen, device="cuda", dtype=torch.float64)
        s["n_acc"], s["next"] = (torch.zeros(R, dtype=torch.int32, device="cuda") for _ in range(2))
        s["p"] = torch.zeros(max(nd, 1), dtype=torch.float32, device="cuda")
        # the plain form's padded draft table
        width = max(max(kk), 1)
        slot = torch.arange(width, device="cuda")
        first = s["row_off"][:-1].long() - torch.arange(R, device="cuda")
        s["slot_kept"] = slot < torch.tensor(kk, device="cuda")[:, None]
        s["slot_draft"] = (first[:, None] + slot).clamp(max=max(nd - 1, 0))
        s["kk"] = torch.tensor(kk, device="cuda")
    return s


# ---- the plain forms ----

def _norm_rope_plain(s):
    n, H, KV, D = s["n"], s["H"], s["KV"], s["D"]
    x = s["qkv"][:, :(H + 2 * KV) * D].float().view(n, H + 2 * KV, D)
    table = s["rope"][s["pos"].long()]
    c, sn = table[:, None, :D // 2], table[:, None, D // 2:]

    def turn(y, w):
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w
        a, b = y[..., :D // 2], y[..., D // 2:]
        return torch.cat([a * c - b * sn, a * sn + b * c], -1)

    q, k = turn(x[:, :H], s["q_norm"]), turn(x[:, H:H + KV], s["k_norm"])
    out = {"q": q.to(s["dt"]), "k": k.to(s["dt"])}
    if s["cache"]:
        for name, y in (("k_held", k), ("v_held", x[:, H + KV:])):
            y = y.transpose(0, 1)
            scale = y.abs().amax(-1, keepdim=True) / 127
            held = torch.round(y / scale) * scale
            out[name] = torch.zeros_like(s[name])
            out[name][:, s["kv_at"].long()] = held.to(torch.bfloat16)
    return out


def _softmax(x):
    x = (x - x.amax(-1, keepdim=True)).exp_()
    return x / x.sum(-1, keepdim=True)


def _prompt_plain(s):
    H, KV, D = s["H"], s["KV"], s["D"]
    S, L = s["row"].shape
    q = s["q"].float()[s["row"]].view(S, L, KV, H // KV, D).permute(0, 2, 3, 1, 4)
    k = s["k"].float()[s["row"]].permute(0, 2, 3, 1)[:, :, None]
    v = s["v"].float()[s["row"]].permute(0, 2, 1, 3)[:, :, None]
    seen = torch.ones(L, L, dtype=torch.bool, device="cuda").tril()
    x = torch.matmul(q * (1.0 / math.sqrt(D)), k).masked_fill_(~seen, -math.inf)
    y = torch.matmul(_softmax(x), v).permute(0, 3, 1, 2, 4).reshape(S, L, H, D)
    s["out"][s["row"][s["held"]]] = y[s["held"]].to(s["dt"])
    return s["out"]


def _shared_plain(s):
    n, H, KV, D, groups = s["n"], s["H"], s["KV"], s["D"], s["n_groups"]
    G, R, T = H // KV, s["n_groups"] * s["reqs"], s["toks"]
    scale = 1.0 / math.sqrt(D)

    def rows(name, at):
        return s[name + "8"][:, at].float() * s[name + "s"][:, at][..., None]  # [KV, *at, D]

    q = s["q"].float().view(n, KV, G, D).transpose(0, 1) * scale  # [KV, n, G, D]
    # scores against the prefix of the token's group, its request's own rows and its ancestors
    pk, pv = rows("k", s["pre_row"]), rows("v", s["pre_row"])
    ok, ov = rows("k", s["own_row"]), rows("v", s["own_row"])
    ak, av = rows("k", s["anc_row"]), rows("v", s["anc_row"])
    a = torch.matmul(q.reshape(KV, groups, -1, D), pk.transpose(-1, -2))
    a = a.masked_fill(~s["pre_kept"][None, :, None, :], -math.inf).view(KV, n, G, -1)
    b = torch.matmul(q.reshape(KV, R, T * G, D), ok.transpose(-1, -2)).view(KV, R, T, G, -1)
    b = b.masked_fill(~s["own_kept"][None, :, :, None, :], -math.inf).view(KV, n, G, -1)
    c = torch.matmul(q, ak.transpose(-1, -2)).masked_fill(~s["anc_kept"][None, :, None, :], -math.inf)
    p = _softmax(torch.cat([a, b, c], -1))
    a, b, c = p.split([a.shape[-1], b.shape[-1], c.shape[-1]], -1)
    y = torch.matmul(a.reshape(KV, groups, -1, a.shape[-1]), pv).reshape(KV, n, G, D)
    y = y + torch.matmul(b.reshape(KV, R, T * G, b.shape[-1]), ov).reshape(KV, n, G, D)
    y = y + torch.matmul(c, av)
    return y.transpose(0, 1).reshape(n, H, D).to(s["dt"])


def _verify_plain(s):
    # in 64 bits: a sum over the whole vocabulary, and draws next to a border
    R, nd, off = s["reqs"], s["nd"], s["row_off"][:-1].long()
    each = torch.arange(R, device="cuda")
    x = s["logits"].double()
    best = x.argmax(-1)
    greedy = s["temp"] <= 0
    T = torch.where(greedy, 1.0, s["temp"].double())[s["row_req"]]
    p = _softmax(x / T[:, None])
    p = torch.where(greedy[s["row_req"]][:, None], (torch.arange(s["V"], device="cuda") == best[:, None]).double(), p)
    if nd:
        d = s["draft"].long()
        pd = p[s["draft_row"]].gather(1, d[:, None]).flatten()
        qd = s["q"].gather(1, d[:, None]).flatten().double() if "q" in s else torch.ones_like(pd)
        qd = torch.where(greedy[s["row_req"]][s["draft_row"]], 1.0, qd)
        ok = (qd > 0) & (s["u"][s["draft_row"]] * qd < pd)
        table = (ok[s["slot_draft"]] & s["slot_kept"]).long().cumprod(-1)
        n_acc = table.sum(-1)
        # a draft is looked at while all before it were accepted
        seen = (torch.arange(table.shape[1], device="cuda") <= n_acc[:, None]) & s["slot_kept"]
        shown = torch.zeros(nd, device="cuda")
        shown[s["slot_draft"][seen]] = pd[s["slot_draft"][seen]].float()
    else:
        n_acc, shown = torch.zeros(R, dtype=torch.long, device="cuda"), s["p"]
    last = p[off + n_acc]
    cut = (n_acc < s["kk"]) & ~greedy
    at = (off - each + n_acc).clamp(max=max(nd - 1, 0))
    if "q" in s:
        q = s["q"][at].double()
    else:
        q = (torch.arange(s["V"], device="cuda") == s["draft"].long()[at][:, None]).double()
    rest = torch.where(cut[:, None], (last - q).clamp(min=0), last)
    rest = torch.where((rest.sum(-1) > 0)[:, None], rest, last)
    total = rest.cumsum(-1)
    u = s["u"][off + n_acc + cut.long()]
    hit = (total >= (u * total[:, -1])[:, None]) & (rest > 0)
    return {"n_acc": n_acc.int(), "next": hit.int().argmax(-1).int(), "p": shown}


# ---- the library's calls ----

def _own(s):
    import malkin_b200 as mk
    t, stream = IDS[s["type"]], torch.cuda.current_stream().cuda_stream

    def at(name):
        return s[name].data_ptr() if name in s else 0

    if s["op"] == "norm_rope":
        n, H, KV, D = s["n"], s["H"], s["KV"], s["D"]
        mk.qk_norm_rope(t, at("qkv"), s["ld"], n, H, KV, D, at("q_norm"), at("k_norm"), EPS, at("rope"), s["n_pos"],
                        at("pos"), at("q_out"), H * D, at("k_out"), KV * D, at("k8"), at("v8"), at("ks"), at("vs"),
                        n if s["cache"] else 0, at("kv_at"), stream=stream)
        out = {"q": s["q_out"], "k": s["k_out"]}
        if s["cache"]:  # the 8-bit rows as the values they stand for
            out["k_held"] = torch.mul(s["k8"], s["ks"][..., None], out=s["k_held"])
            out["v_held"] = torch.mul(s["v8"], s["vs"][..., None], out=s["v_held"])
        return out
    if s["op"] == "prompt":
        H, KV, D = s["H"], s["KV"], s["D"]
        mk.attention_prompt(t, at("q"), H * D, at("k"), KV * D, at("v"), KV * D, s["n"], s["n_seq"], at("off"), H, KV,
                            D, 1.0 / math.sqrt(D), at("out"), H * D, stream=stream)
        return s["out"]
    if s["op"] == "shared":
        n, H, KV, D = s["n"], s["H"], s["KV"], s["D"]
        if "ws" not in s:
            s["ws"] = torch.empty(mk.attention_shared_workspace(n, H, KV, D, s["n_groups"]), dtype=torch.uint8,
                                  device="cuda")
        mk.attention_shared(t, at("q"), H * D, n, H, KV, D, 1.0 / math.sqrt(D), at("k8"), at("v8"), at("ks"), at("vs"),
                            s["n_rows"], s["n_groups"], at("group_off"), at("prefix_base"), at("prefix_len"),
                            at("kv_base"), at("n_keys"), at("anc_off"), at("anc"), s["anc"].numel(), at("out"), H * D,
                            at("ws"), s["ws"].numel(), stream=stream)
        return s["out"]
    if "ws" not in s:
        s["ws"] = torch.empty(mk.verify_draft_workspace(s["m"], s["reqs"], s["V"]), dtype=torch.uint8, device="cuda")
    mk.verify_draft(t, at("logits"), s["V"], s["m"], s["V"], s["reqs"], at("row_off"), at("draft"), at("q"), s["V"],
                    at("temp"), at("u"), at("n_acc"), at("next"), at("p"), at("ws"), s["ws"].numel(), stream=stream)
    return {"n_acc": s["n_acc"], "next": s["next"], "p": s["p"]}


def run(state):
    if own:
        return _own(state)
    return {"norm_rope": _norm_rope_plain, "prompt": _prompt_plain, "shared": _shared_plain,
            "verify": _verify_plain}[state["op"]](state)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "verify":
        # every row of logits, and of each request the one row of draft probabilities that its residual needs
        rows = sum(_lengths(case)) + case["reqs"]
        return {"bytes": rows * case["V"] * size + (case["reqs"] * case["V"] * 4 if case["probs"] else 0),
                "flops": 4 * rows * case["V"]}
    H, KV, D = case["H"], case["KV"], case["D"]
    if case["op"] == "norm_rope":
        n = case["n"]
        bytes_ = n * (2 * (H + KV) * D * size + D * 4 + 4)
        if case["cache"]:
            bytes_ += n * KV * (D * size + 2 * (D + 4))
        return {"bytes": bytes_, "flops": n * (H + KV) * D * 8}
    if case["op"] == "prompt":
        lens = _lengths(case)
        return {"bytes": sum(lens) * (2 * H + 2 * KV) * D * size, "flops": sum(2 * x * (x + 1) for x in lens) * H * D}
    prefix, owned = _lengths(case)
    T = case["toks"]
    n = len(owned) * T
    rows = sum(prefix) + sum(owned) + n
    pairs = T * (case["reqs"] * sum(prefix) + sum(owned)) + len(owned) * T * (T + 1) / 2
    return {"bytes": rows * KV * 2 * (D + 4) + 2 * n * H * D * size, "flops": 4 * H * D * pairs}


# ---- 64 bits, from the definitions ----

def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "norm_rope":
        n, H, KV, D = case["n"], case["H"], case["KV"], case["D"]
        out = {"q": torch.empty(n, H, D, dtype=f, device="cuda"), "k": torch.empty(n, KV, D, dtype=f, device="cuda")}
        spin = torch.complex(s["rope"][:, :D // 2].to(f), s["rope"][:, D // 2:].to(f))[s["pos"].long()]
        heads = s["qkv"][:, :(H + 2 * KV) * D].to(f).reshape(n, -1, D)
        for h in range(H + KV):
            x = heads[:, h]
            x = x / torch.sqrt((x * x).sum(1) / D + EPS)[:, None] * (s["q_norm"] if h < H else s["k_norm"]).to(f)
            z = torch.complex(x[:, :D // 2].contiguous(), x[:, D // 2:].contiguous()) * spin
            (out["q"][:, h] if h < H else out["k"][:, h - H])[:] = torch.cat([z.real, z.imag], 1)
        if case["cache"]:
            for name, x in (("k_held", out["k"]), ("v_held", heads[:, H + KV:])):
                step = x.abs().amax(2, keepdim=True) / 127
                out[name] = torch.zeros(KV, n, D, dtype=f, device="cuda")
                out[name][:, s["kv_at"].long()] = (torch.round(x / step) * step).transpose(0, 1)
        return out
    if case["op"] == "prompt":
        H, KV, D = case["H"], case["KV"], case["D"]
        out = torch.zeros(s["n"], H, D, dtype=f, device="cuda")
        lo = 0
        for length in s["lens"]:
            hi = lo + length
            later = torch.arange(length, device="cuda")[:, None] < torch.arange(length, device="cuda")
            for h in range(H):
                kv = h // (H // KV)
                x = s["q"][lo:hi, h].to(f) @ s["k"][lo:hi, kv].to(f).T / math.sqrt(D)
                x[later] = -math.inf
                x -= torch.logsumexp(x, 1, keepdim=True)
                out[lo:hi, h] = x.exp_() @ s["v"][lo:hi, kv].to(f)
            lo = hi
        return out
    if case["op"] == "shared":
        H, KV, D, T = case["H"], case["KV"], case["D"], case["toks"]
        G, n = H // KV, s["n"]
        out = torch.zeros(n, H, D, dtype=f, device="cuda")
        base, keys, a_off = s["kv_base"].tolist(), s["n_keys"].tolist(), s["anc_off"].tolist()
        p_base, p_len = s["prefix_base"].tolist(), s["prefix_len"].tolist()
        for t0 in range(0, n, T):
            g = t0 // (T * case["reqs"])
            # every row that one of the request's tokens looks at, then who looks at which
            own_n = max(keys[t0:t0 + T])
            extra = s["anc"][a_off[t0]:a_off[t0 + T]].long() + base[t0]
            look = torch.cat([torch.arange(p_base[g], p_base[g] + p_len[g], device="cuda"),
                              torch.arange(base[t0], base[t0] + own_n, device="cuda"), extra])
            hidden = torch.zeros(T, look.numel(), dtype=torch.bool, device="cuda")
            for i in range(T):
                hidden[i, p_len[g] + keys[t0 + i]:] = True
                lo = p_len[g] + own_n - a_off[t0]
                hidden[i, lo + a_off[t0 + i]:lo + a_off[t0 + i + 1]] = False
            for kv in range(KV):
                k = s["k8"][kv, look].to(f) * s["ks"][kv, look].to(f)[:, None]
                v = s["v8"][kv, look].to(f) * s["vs"][kv, look].to(f)[:, None]
                x = torch.einsum("tgd,jd->tgj", s["q"][t0:t0 + T, kv * G:(kv + 1) * G].to(f), k) / math.sqrt(D)
                x = x.masked_fill(hidden[:, None], -math.inf)
                out[t0:t0 + T, kv * G:(kv + 1) * G] = torch.softmax(x, -1) @ v
        return out
    off, temp = s["row_off"].tolist(), s["temp"].tolist()
    n_acc, nxt, shown = [], [], torch.zeros(max(s["nd"], 1), dtype=f, device="cuda")
    for r in range(case["reqs"]):
        k, i, token = off[r + 1] - off[r] - 1, 0, None
        while token is None:
            row = s["logits"][off[r] + i].to(f)
            if temp[r] > 0:
                p = torch.exp(torch.log_softmax(row / s["temp"][r].to(f), 0))
            else:
                p = torch.zeros_like(row)
                p[torch.nonzero(row == row.max())[0, 0]] = 1
            left = p
            if i < k:
                j = off[r] - r + i
                d = int(s["draft"][j])
                shown[j] = p[d]
                if temp[r] <= 0:
                    taken = bool(p[d] == 1)
                else:
                    q = s["q"][j].to(f) if case["probs"] else torch.nn.functional.one_hot(torch.tensor(d), case["V"]).to(f).cuda()
                    taken = bool(q[d] > 0) and bool(s["u"][off[r] + i] * q[d] < p[d])
                    left = torch.relu(p - q)
                    left = left if float(left.sum()) > 0 else p
                if taken:
                    i += 1
                    continue
            some = torch.nonzero(left > 0).flatten()
            run_ = torch.cumsum(left[some], 0)
            u = s["u"][off[r] + i + (1 if i < k and temp[r] > 0 else 0)]
            token = int(some[min(int(torch.searchsorted(run_, u * run_[-1])), some.numel() - 1)])
        n_acc.append(i)
        nxt.append(token)
    return {"n_acc": _ints(n_acc), "next": _ints(nxt), "p": shown}
