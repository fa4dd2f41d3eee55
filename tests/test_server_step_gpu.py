"""A small decoder served to several sequences with 8-bit linears over the paged 4-bit cache: prompts, forks that share a
prompt, decode steps and sampled tokens, every operator's output against 64 bits on the inputs it got."""
import math

import numpy as np
import pytest
import torch

import kv4_ref as R
from soinfer import ops
from soinfer.quant import formats
from soinfer.runtime.paged_kv import PagedKV4
from test_int8_gpu import check_gate_up, check_linear, check_rows, rows_ref
from test_sample_gpu import reference as sample_reference

pytestmark = pytest.mark.gpu
H, NQ, NKV, HD, I, V, LAYERS, PAGE, GS = 256, 8, 2, 64, 528, 1003, 2, 16, 32


class Server:
    """check=True compares each operator's output; the calls are the same either way."""

    def __init__(self, dev, seed):
        g = torch.Generator(device=dev).manual_seed(seed)

        def weight(n, k):
            qt = formats.quantize(torch.randn(n, k, generator=g, device=dev) / math.sqrt(k), formats.QuantConfig(8, "per_channel"))
            return qt.qweight, qt.scale

        def norm(n):
            return (1 + 0.1 * torch.randn(n, generator=g, device=dev)).half()

        self.embed = torch.randn(V, H, generator=g, device=dev).half()
        self.layers = [dict(n1=norm(H), n2=norm(H), qn=norm(HD), kn=norm(HD), qkv=weight((NQ + 2 * NKV) * HD, H), o=weight(H, NQ * HD),
                            gate=weight(I, H), up=weight(I, H), down=weight(H, I)) for _ in range(LAYERS)]
        self.norm, self.head = norm(H), weight(V, H)
        self.cos, self.sin = (torch.from_numpy(x).to(dev) for x in R.rope_tables(600, HD))
        self.cache = PagedKV4(LAYERS, 120, NKV, HD, max_len=600, group_size=GS, page_size=PAGE, device=dev)
        self.check = True
        self.shared_calls = 0

    def linear(self, x, xs, w, residual=None):
        y = ops.int8_linear(x, xs, *w, residual=residual)
        if self.check:
            check_linear(y, x, xs, *w, residual)
        return y

    def quantized(self, x, weight=None):
        q, s = ops.quantize_int8(x, weight)
        if self.check:
            check_rows((q, s), rows_ref(x, None, weight, 1e-6))
        return q, s

    def attend(self, layer, step, q):
        out = self.cache.attend(layer, step, q)
        self.shared_calls += step.cu_groups is not None
        if self.check:
            k, v, cu = self.cache.read(layer, step)  # rounded to binary16, which moves a score by 2^-11 sum |q k| scale
            for i in range(len(step.sequences)):
                at = slice(int(cu[i]), int(cu[i + 1]))
                kb, vb = k[at].double(), v[at].double()
                ref, bound = R.attention(q[i:i + 1].double(), kb, vb, torch.tensor([len(kb) - 1], device=q.device), 1 / math.sqrt(HD))
                for h in range(NQ):
                    kh, vh = kb[:, h * NKV // NQ], vb[:, h * NKV // NQ]
                    d = 2.0 ** -11 * (q[i, h].double().abs() @ kh.abs().T).amax() / math.sqrt(HD)
                    bound[0, h] += (2 * d + 2.0 ** -11) * vh.abs().amax(0)
                R.assert_within(out[i:i + 1], ref, bound, f"layer {layer} sequence {i}")
        return out

    def forward(self, step, tokens, prompt):
        """The last rows' logits: of every row in a decode step, of each sequence's last one in a prompt."""
        h = self.embed[tokens.long()]
        T = h.shape[0]
        q, s = self.quantized(h, self.layers[0]["n1"])
        for i, w in enumerate(self.layers):
            qkv = self.linear(q, s, w["qkv"])
            if prompt:
                qr, k = self.cache.append(i, step, qkv, w["qn"], w["kn"], self.cos, self.sin, NQ, keep_k=True)
                o = self.cache.prompt(i, step, qr, k, qkv.view(T, -1, HD)[:, NQ + NKV:])
            else:
                o = self.attend(i, step, self.cache.append(i, step, qkv, w["qn"], w["kn"], self.cos, self.sin, NQ))
            o = self.linear(*self.quantized(o.view(T, NQ * HD)), w["o"])
            q, s, h2 = ops.add_rmsnorm_int8(o, h, w["n2"])
            if self.check:
                ref = rows_ref(o, h, w["n2"], 1e-6)
                check_rows((q, s), ref)
                assert torch.equal(h2, ref[3])
            g = ops.int8_gate_up(q, s, *w["gate"], *w["up"])
            if self.check:
                check_gate_up(g, q, s, [w["gate"][0], w["up"][0]], [w["gate"][1], w["up"][1]])
            h = self.linear(*self.quantized(g), w["down"], residual=h2)
            q, s = self.quantized(h, self.layers[i + 1]["n1"] if i + 1 < LAYERS else self.norm)
        if prompt:
            last = (step.cu_seqlens[1:] - 1).long()
            q, s = q[last], s[last]
        return self.linear(q, s, self.head)

    def sample(self, logits, u, T=0.8, k=50, p=0.95, m=0.01):
        got = ops.sample_tokens(logits, u, T, k, p, m)
        if self.check:
            for b in range(len(u)):
                _, also = sample_reference(logits[b].float().cpu().numpy(), u[b].item(), T, k, p, m)
                assert int(got[b]) in also
        return got


def test_prompts_forks_and_sampled_steps(cuda):
    server = Server(cuda, 1)
    c = server.cache
    g = torch.Generator(device=cuda).manual_seed(2)
    a, b = c.add(), c.add()
    step = c.step({a: 133, b: 37})
    first = server.sample(server.forward(step, torch.randint(0, V, (170,), generator=g, device=cuda), True),
                          torch.rand(2, generator=g, device=cuda))
    assert server.shared_calls == 0
    forks = [c.fork(a) for _ in range(3)]  # 128 tokens each, the prompt's last five are appended again below
    order = [a, *forks, b]
    tokens = torch.cat([first[:1].expand(4), first[1:]])
    seen = set()
    for _ in range(3):
        step = c.step({s: 1 for s in order})
        tokens = server.sample(server.forward(step, tokens, False), torch.rand(5, generator=g, device=cuda))
        seen.add(tuple(tokens.tolist()))
        assert step.cu_groups.tolist() == [0, 4, 5] and step.shared_lens.tolist() == [128] * 4 + [0]
    assert server.shared_calls == 3 * LAYERS and len(seen) == 3
    for s in (a, *forks[:2]):
        c.free(s)
    step = c.step({forks[2]: 1, b: 1})
    assert step.cu_groups is None
    server.forward(step, tokens[:2], False)


def test_a_captured_step(cuda):
    """A decode step recorded once: replays with other tokens, positions and random numbers give the eager step's tokens."""
    server = Server(cuda, 3)
    c = server.cache
    server.check = False
    g = torch.Generator(device=cuda).manual_seed(4)
    a = c.add()
    server.forward(c.step({a: 150}), torch.randint(0, V, (150,), generator=g, device=cuda), True)
    seqs = [a, c.fork(a), c.fork(a)]
    step = c.step({s: 1 for s in seqs})
    tokens, u = torch.zeros(3, dtype=torch.int32, device=cuda), torch.zeros(3, device=cuda)
    step.max_len = 320  # (the longest that a replay may reach: the table below has room for it)
    tables = step.block_table
    step.block_table = torch.zeros(3, 20, dtype=torch.int32, device=cuda)
    step.block_table[:, :tables.shape[1]] = tables
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        server.sample(server.forward(step, tokens, False), u)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = server.sample(server.forward(step, tokens, False), u)
    for _ in range(4):
        now = c.step({s: 1 for s in seqs})
        step.block_table.zero_()
        step.block_table[:, :now.block_table.shape[1]] = now.block_table
        step.seq_lens.copy_(now.seq_lens)
        tokens.copy_(torch.randint(0, V, (3,), generator=g, device=cuda))
        u.copy_(torch.rand(3, generator=g, device=cuda))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        now.max_len, now.block_table = step.max_len, step.block_table  # (the same bounds: the same splits)
        want = server.sample(server.forward(now, tokens, False), u)  # writes the same rows again
        assert torch.equal(got, want)


def test_two_streams_at_once(cuda):
    """Two servers whose steps overlap on two streams give what each gives alone."""
    servers, inputs, want = [], [], []
    for i in range(2):
        s = Server(cuda, 10 + i)
        s.check = False
        g = torch.Generator(device=cuda).manual_seed(i)
        a = s.cache.add()
        s.forward(s.cache.step({a: 100 + 60 * i}), torch.randint(0, V, (100 + 60 * i,), generator=g, device=cuda), True)
        seqs = [a] + [s.cache.fork(a) for _ in range(4)]
        step = s.cache.step({x: 1 for x in seqs})
        tokens, u = torch.randint(0, V, (5,), generator=g, device=cuda), torch.rand(5, generator=g, device=cuda)
        servers.append(s)
        inputs.append((step, tokens, u))
        want.append(s.sample(s.forward(step, tokens, False), u))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                step, tokens, u = inputs[i]
                got[i].append(servers[i].sample(servers[i].forward(step, tokens, False), u))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
