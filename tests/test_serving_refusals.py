"""Refusals of the serving operators: every one is made before a device is looked at, so they are tested without a GPU."""
import pytest

F32, F16, BF16, Q8 = 0, 1, 30, 8
P = 1 << 20  # stands for a device pointer: the calls below are refused before it is looked at


def refused(mk, f, *a, code=None, text=None, **k):
    with pytest.raises(mk.MalkinError) as e:
        f(*a, **k)
    assert e.value.code == (mk.MK_ERR_ARG if code is None else code), str(e.value)
    if text:
        assert text in str(e.value)


def norm(mk, **k):
    a = dict(type_=BF16, dev_qkv=P, ld=6 * 128, n=2, H=2, KV=2, D=128, dev_q_norm=P, dev_k_norm=P, eps=1e-6, dev_rope=P,
             n_pos=4, dev_pos=P, dev_q=P, q_ld=256, dev_k=P, k_ld=256)
    a.update(k)
    mk.qk_norm_rope(**a)


@pytest.mark.parametrize("change", [
    dict(type_=Q8), dict(type_=99), dict(n=-1), dict(H=0), dict(KV=0), dict(H=5000), dict(D=96), dict(D=0),
    dict(n_pos=0), dict(eps=-1.0), dict(eps=float("nan")), dict(ld=6 * 128 - 1), dict(q_ld=255), dict(k_ld=255),
    dict(dev_kc=P, dev_vc=P, dev_ks=P, dev_vs=P, n_rows=0, dev_kv_at=P),
    dict(dev_kc=P, dev_vc=P, dev_ks=P, dev_vs=P, n_rows=4), dict(dev_kc=P, n_rows=4, dev_kv_at=P),
    dict(dev_qkv=0), dict(dev_qkv=P + 1), dict(dev_pos=P + 2), dict(dev_q=0), dict(type_=F32, dev_q=P + 2)])
def test_norm_rope_refuses(mk, change):
    refused(mk, norm, mk, **change)


def prompt(mk, **k):
    a = dict(type_=BF16, dev_q=P, q_ld=512, dev_k=P, k_ld=256, dev_v=P, v_ld=256, n=10, n_seq=2, dev_off=P, H=4, KV=2,
             D=128, scale=0.1, dev_out=P, out_ld=512)
    a.update(k)
    mk.attention_prompt(**a)


@pytest.mark.parametrize("change", [
    dict(type_=F32), dict(type_=Q8), dict(H=0), dict(KV=0), dict(H=3), dict(D=96), dict(n=-1), dict(n_seq=-1),
    dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(q_ld=511),
    dict(q_ld=516), dict(k_ld=255), dict(v_ld=260), dict(out_ld=504), dict(dev_q=P + 8), dict(dev_out=P + 2),
    dict(dev_k=0), dict(dev_off=P + 1)])
def test_prompt_refuses(mk, change):
    refused(mk, prompt, mk, **change)


def test_prompt_width_256_is_unsupported(mk):
    refused(mk, prompt, mk, D=256, q_ld=1024, k_ld=512, v_ld=512, out_ld=1024, code=mk.MK_ERR_UNSUPPORTED)


def shared(mk, **k):
    a = dict(type_=F16, dev_q=P, q_ld=512, n=6, H=4, KV=2, D=128, scale=0.1, dev_k=P, dev_v=P, dev_ks=P, dev_vs=P,
             n_rows=100, n_groups=1, dev_group_off=P, dev_prefix_base=P, dev_prefix_len=P, dev_kv_base=P, dev_n_keys=P,
             dev_anc_off=P, dev_anc=P, n_anc=3, dev_out=P, out_ld=512, dev_ws=P, ws_bytes=1 << 40)
    a.update(k)
    mk.attention_shared(**a)


@pytest.mark.parametrize("change", [
    dict(type_=F32), dict(H=5), dict(H=0), dict(D=80), dict(n=-1), dict(n_groups=-1), dict(n_rows=0), dict(n_anc=-1),
    dict(H=258, KV=2, q_ld=258 * 128, out_ld=258 * 128), dict(scale=0.0), dict(scale=float("nan")), dict(q_ld=508),
    dict(q_ld=515), dict(out_ld=511), dict(dev_q=P + 8), dict(dev_k=P + 4), dict(dev_out=P + 4), dict(dev_ws=P + 8),
    dict(dev_ws=P + 16), dict(dev_ks=0), dict(dev_group_off=0), dict(dev_kv_base=0), dict(dev_n_keys=P + 1), dict(dev_anc=0)])
def test_shared_refuses(mk, change):
    refused(mk, shared, mk, **change)


def test_shared_width_256_is_unsupported(mk):
    refused(mk, shared, mk, D=256, q_ld=1024, out_ld=1024, code=mk.MK_ERR_UNSUPPORTED)
    refused(mk, mk.attention_shared_workspace, 4, 4, 2, 256, 1, code=mk.MK_ERR_UNSUPPORTED)
    refused(mk, mk.attention_shared_workspace, 4, 3, 2, 128, 1)
    refused(mk, mk.attention_shared_workspace, -4, 4, 2, 128, 1)


def verify(mk, **k):
    a = dict(type_=F32, dev_logits=P, ld=100, n_rows=6, V=100, n_req=2, dev_row_off=P, dev_draft=P, dev_q=P, q_ld=100,
             dev_temperature=P, dev_uniforms=P, dev_n_acc=P, dev_next=P, dev_p=P, dev_ws=P, ws_bytes=1 << 20)
    a.update(k)
    mk.verify_draft(**a)


@pytest.mark.parametrize("change", [
    dict(type_=Q8), dict(V=0), dict(V=(1 << 27) + 1, ld=1 << 28, q_ld=1 << 28), dict(n_req=-1), dict(n_rows=1),
    dict(ld=99), dict(q_ld=99), dict(ws_bytes=0), dict(dev_ws=P + 8), dict(dev_logits=0), dict(dev_logits=P + 2),
    dict(dev_uniforms=P + 4), dict(dev_row_off=0), dict(dev_draft=0), dict(dev_next=0)])
def test_verify_refuses(mk, change):
    refused(mk, verify, mk, **change)


def test_workspace_sizes(mk):
    assert mk.verify_draft_workspace(0, 0, 1) > 0
    assert mk.verify_draft_workspace(9, 1, 151936) >= 9 * 38 * 16
    refused(mk, mk.verify_draft_workspace, 1, 1, 0)
    refused(mk, mk.verify_draft_workspace, -1, 0, 10)


def test_nothing_to_do(mk):
    """No tokens, no requests: nothing is looked at."""
    norm(mk, n=0)
    verify(mk, n_req=0, n_rows=0)
    prompt(mk, n=0)
    prompt(mk, n_seq=0)
    shared(mk, n=0)
