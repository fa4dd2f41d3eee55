"""PagedKV4: its book-keeping on the CPU, and prompts, decode steps and a continued prompt strung together on the GPU,
against the 64-bit attention over what the cache holds."""
import math

import pytest
import torch

import kv4_ref as R


def make(**kw):
    from soinfer.runtime.paged_kv import PagedKV4

    args = dict(layers=2, num_pages=6, num_kv_heads=2, head_dim=64, max_len=64, group_size=32, page_size=16, device="cpu") | kw
    return PagedKV4(**args)


def test_pages_are_handed_out_and_given_back():
    c = make()
    a, b = c.add(), c.add()
    s = c.step({a: 17, b: 1})
    assert c.free_pages == 3 and s.lens == (17, 1) and s.tokens == 18 and s.max_new == 17 and s.max_len == 17
    assert s.cu_seqlens.tolist() == [0, 17, 18] and s.seq_lens.tolist() == [17, 1] and s.block_table.shape == (2, 2)
    used = {s.block_table[0, 0].item(), s.block_table[0, 1].item(), s.block_table[1, 0].item()}
    assert len(used) == 3
    s = c.step({b: 15})
    assert c.free_pages == 3 and s.block_table.shape == (1, 1) and c.length(b) == 16
    c.step({b: 1, a: 0})
    assert c.free_pages == 2 and c.length(a) == 17
    c.free(a)
    assert c.free_pages == 4
    with pytest.raises(KeyError):
        c.step({a: 1})


def test_a_step_that_does_not_fit_changes_nothing():
    c = make()
    a, b = c.add(), c.add()
    c.step({a: 40})
    with pytest.raises(RuntimeError, match="pages needed"):
        c.step({a: 5, b: 60})
    with pytest.raises(RuntimeError, match="max_len"):
        c.step({b: 1, a: 25})
    assert c.length(a) == 40 and c.length(b) == 0 and c.free_pages == 3
    for bad in ({}, {a: -1}):
        with pytest.raises(ValueError):
            c.step(bad)


@pytest.mark.parametrize("bad", [dict(head_dim=96), dict(group_size=128), dict(group_size=16), dict(page_size=24),
                                 dict(page_size=8), dict(layers=0), dict(num_pages=0), dict(max_len=0)], ids=str)
def test_refused_shapes(bad):
    with pytest.raises(ValueError):
        make(**bad)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,gs,page", [(128, 64, 64), (64, 32, 16)])
def test_prompts_steps_and_a_continued_prompt(cuda, hd, gs, page):
    NQ, NKV, layers = 6, 2, 2
    g = torch.Generator(device=cuda).manual_seed(hd)
    cache = make(layers=layers, num_pages=60 * 64 // page, num_kv_heads=NKV, head_dim=hd, max_len=600, group_size=gs,
                 page_size=page, device=cuda)
    cos, sin = (torch.from_numpy(x).to(cuda) for x in R.rope_tables(600, hd))
    w = [(1 + 0.2 * torch.randn(hd, generator=g, device=cuda)).half() for _ in range(2)]
    held = {}  # (layer, sequence) -> what the cache holds, 64 bits

    def rows(n):
        return torch.randn((n, (NQ + 2 * NKV) * hd), generator=g, device=cuda).half()

    def check(out, q, layer, step, keys, label):
        at = 0
        for i, s in enumerate(step.sequences):
            n = step.new[i]
            k, v = keys[layer, s]
            ref, bound = R.attention(q[at:at + n].double(), k, v, torch.arange(n, device=cuda) + len(k) - n, 1 / math.sqrt(hd))
            R.assert_within(out[at:at + n], ref, bound, f"{label} layer {layer} sequence {s}")
            at += n

    def enter(step, keep_k):
        out = {}
        for layer in range(layers):
            qkv = rows(step.tokens)
            got = cache.append(layer, step, qkv, *w, cos, sin, NQ, keep_k=keep_k)
            k, v, cu_k = cache.read(layer, step)
            for i, s in enumerate(step.sequences):
                at = slice(int(cu_k[i]), int(cu_k[i + 1]))
                now = (k[at].double(), v[at].double())
                if (layer, s) in held:  # what was there has not changed
                    n = len(held[layer, s][0])
                    assert torch.equal(held[layer, s][0], now[0][:n]) and torch.equal(held[layer, s][1], now[1][:n])
                held[layer, s] = now
            out[layer] = (qkv, got)
        return out

    a, b, c = cache.add(), cache.add(), cache.add()
    step = cache.step({a: 130, b: 1, c: 77})
    own = {}
    for layer, (qkv, (q, k)) in enter(step, True).items():
        v = qkv.view(-1, NQ + 2 * NKV, hd)[:, NQ + NKV:]
        at = 0
        for s, n in zip(step.sequences, step.new):
            own[layer, s] = (k[at:at + n].double(), v[at:at + n].double())
            # the cache holds these rows to half a step of their group, with the scale's and the value's rounding
            for x, y in zip(held[layer, s], own[layer, s]):
                top = y.unflatten(-1, (-1, gs)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, gs).flatten(-2)
                assert ((x - y).abs() <= top / 14 * (1 + 2 ** -9) + y.abs() * 2 ** -10).all()
            at += n
        check(cache.prompt(layer, step, q, k, v), q, layer, step, own, "prompt")
    for _ in range(3):  # decode steps, in another order of the sequences
        step = cache.step({c: 1, a: 1, b: 1})
        for layer, (_, q) in enter(step, False).items():
            got = cache.attend(layer, step, q)
            # the attention multiplies by code and scale, the read rounds their product: half a binary16 step of v, and of
            # each k a relative 2^-11, which moves a score by up to 2^-11 sum |q k| scale
            for i, s in enumerate(step.sequences):
                k, v = held[layer, s]
                ref, bound = R.attention(q[i:i + 1].double(), k, v, torch.tensor([len(k) - 1], device=cuda), 1 / math.sqrt(hd))
                rep = NQ // NKV
                for h in range(NQ):
                    kh, vh = k[:, h // rep], v[:, h // rep]
                    d = 2.0 ** -11 * (q[i, h].double().abs() @ kh.abs().T).amax() / math.sqrt(hd)
                    bound[0, h] += (2 * d + 2.0 ** -11) * vh.abs().amax(0)
                R.assert_within(got[i:i + 1], ref, bound, f"decode layer {layer} sequence {s}")
    cache.free(b)
    step = cache.step({a: 50, c: 300})  # prompts that continue a context: their keys are read back from the pages
    for layer, (_, q) in enter(step, False).items():
        check(cache.prompt(layer, step, q), q, layer, step, held, "continued")
    with pytest.raises(ValueError, match="begin"):
        cache.prompt(0, step, q, k, v)
