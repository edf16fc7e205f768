"""Serving with the 8-bit cache and the drawn tokens together: ragged prompts, then steps
replayed from one captured graph, on the blocks of a GPT-2; and generate's drawn tokens."""

import pytest
import torch

import cutilegpt_amd as cg
from paged8_ref import F8
from sample_ref import draw

pytestmark = pytest.mark.gpu

F32, I8 = torch.float32, torch.int8


class Server:
    """GPT-2 blocks over pools of 8-bit pages; ``check`` reads every layer's cache back and runs
    the 32-bit paged attention on it instead."""

    def __init__(self, model, code, gpu, n_pages=40, page=16, block=8):
        cfg = model.config
        self.model, self.H, self.hd, self.page = model, cfg.n_head, cfg.head_dim, page
        shape = (cfg.n_layer, 2, n_pages, self.H, page)
        self.pools = torch.zeros(*shape, self.hd, dtype=torch.uint8, device=gpu).view(code)
        self.scales = torch.zeros(*shape[:-1], page // block, dtype=torch.uint8, device=gpu)
        self.n_pages = n_pages

    def forward(self, tokens, pos, table, lens, cu=None, check=None):
        W, H, hd = self.model.weights, self.H, self.hd
        x = W["wte"][tokens] + W["wpe"][pos]  # (no copy to the host: the step is captured)
        for i in range(self.model.config.n_layer):
            w = lambda n: W[f"h.{i}.{n}"]
            h = cg.cutile_layer_norm(x, w("ln_1.weight"), w("ln_1.bias"))
            qkv = cg.cutile_linear_bias(h, w("attn.c_attn.weight"), w("attn.c_attn.bias")).view(-1, 3 * H, hd)
            q, k, v = qkv[:, :H], qkv[:, H:2 * H], qkv[:, 2 * H:]
            cache = self.pools[i, 0], self.pools[i, 1], self.scales[i, 0], self.scales[i, 1], table, lens
            cg.paged_kv_append_8bit(k, v, *cache, cu_q=cu)
            a = cg.paged_attention_8bit(q, *cache, cu_q=cu)
            if check is not None:
                n = int(lens.sum())
                rows = torch.cat([torch.zeros_like(lens[:1]), lens.cumsum(0, dtype=torch.int32)])
                kr, vr = cg.paged_kv_read_8bit(*cache, rows, n, F32)
                wide = [torch.zeros(self.n_pages, H, self.page, hd, device=x.device) for _ in range(2)]
                cg.paged_kv_append(kr, vr, *wide, table, lens, cu_q=rows)
                b = cg.paged_attention(q, *wide, table, lens, cu_q=cu)
                check.append((a - b).abs().max())
            x = x + cg.cutile_linear_bias(a.view(-1, H * hd), w("attn.c_proj.weight"), w("attn.c_proj.bias"))
            h = cg.cutile_layer_norm(x, w("ln_2.weight"), w("ln_2.bias"))
            x = x + cg.cutile_fused_mlp(h, w("mlp.c_fc.weight"), w("mlp.c_fc.bias"), w("mlp.c_proj.weight"),
                                        w("mlp.c_proj.bias"))
        x = cg.cutile_layer_norm(x, W["ln_f.weight"], W["ln_f.bias"])
        return cg.cutile_linear(x, W["lm_head.weight"])


@pytest.mark.parametrize("code", [F8, I8])
def test_serving(gpu, code):
    cfg = cg.GPTConfig.gpt_nano()
    model = cg.CutileGPT(cfg, dtype=F32, seed=3)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in (37, 5, 60)]
    B, steps = 3, 8
    table = torch.randperm(40, generator=g)[:B * 8].view(B, 8).to(gpu, torch.int32)
    u = torch.rand(steps + 1, B, generator=g)
    settings = dict(temperature=0.9, top_k=50, top_p=0.95, min_p=0.001)
    names = dict(T=0.9, k=50, p=0.95, m=0.001)
    lens = torch.tensor([len(s) for s in prompts], dtype=torch.int32, device=gpu)
    cu = torch.tensor([0, 37, 42, 102], dtype=torch.int32, device=gpu)
    last = cu[1:].long() - 1
    pos = torch.cat([torch.arange(len(s)) for s in prompts]).to(gpu)

    def drawn(logits, got, t):
        # The kernel's token is the float64 draw from the same logits, with near certainty.
        for b in range(B):
            want, margin = draw(logits[b].cpu(), float(u[t, b]), **names)
            assert int(got[b]) == want or margin < 1e-8, (t, b)

    # Eagerly, every layer beside the 32-bit attention over the same values.
    eager, off = Server(model, code, gpu), []
    logits = eager.forward(torch.cat(prompts).to(gpu), pos, table, lens, cu, check=off)
    # (The prompts' forward in full precision: the 8 bits move the logits, but not out of sight.)
    for b, s in enumerate(prompts):
        want = model(s[None].to(gpu))[0][0]
        assert (logits[int(cu[b]):int(cu[b + 1])] - want).abs().max() < 0.1 * want.abs().max()
    after = eager.pools.clone(), eager.scales.clone()
    first = cg.sample_tokens(logits[last], u[0].to(gpu), **settings)
    drawn(logits[last], first, 0)
    tokens, want, el = first, [], lens.clone()
    for t in range(steps):
        el += 1
        logits = eager.forward(tokens, el.long() - 1, table, el, check=off)
        tokens = cg.sample_tokens(logits, u[t + 1].to(gpu), **settings)
        drawn(logits, tokens, t + 1)
        want.append(tokens)
    # Outputs of order 1; both sides hold what fp32 does.
    assert max(float(x) for x in off) < 1e-5

    # The steps from one graph: tokens, lengths and numbers stay on the device.
    served = Server(model, code, gpu)
    served.pools, served.scales = after
    spare = Server(model, code, gpu)
    ids, sl, uu = first.clone(), lens + 1, u[1].to(gpu)

    def step(server):
        out = server.forward(ids, sl.long() - 1, table, sl)
        cg.sample_tokens(out, uu, **settings, out=ids)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(spare)
    torch.cuda.current_stream().wait_stream(side)
    ids.copy_(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(served)
    for t in range(steps):
        uu.copy_(u[t + 1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ids, want[t]), t
        sl += 1
    for a, b in ((served.pools.view(torch.uint8), eager.pools.view(torch.uint8)), (served.scales, eager.scales)):
        assert torch.equal(a, b)


def test_generate_draws(gpu):
    """generate with top_p, min_p or a generator draws what sample_tokens draws from its logits;
    with or without the cache and the graph the same tokens come out."""
    cfg = cg.GPTConfig.gpt_nano()
    model = cg.CutileGPT(cfg, dtype=F32, seed=5)
    idx = torch.randint(0, cfg.vocab_size, (3, 9), generator=torch.Generator().manual_seed(1)).to(gpu)
    n = 10
    for kw in (dict(top_p=0.9), dict(temperature=0.7, top_k=20, min_p=0.01), dict(temperature=1.3, top_k=5, top_p=0.8, min_p=0.05), dict()):
        seed = lambda: torch.Generator(device=gpu).manual_seed(7)
        u = torch.rand(n, 3, device=gpu, generator=seed())
        got = [model.generate(idx, n, generator=seed(), use_cache=c, use_graph=r, **kw) for c, r in ((True, True), (True, False), (False, False))]
        seq = idx
        for t in range(n):
            logits = model(seq)[0][:, -1]
            nxt = cg.sample_tokens(logits, u[t], **kw)
            seq = torch.cat([seq, nxt[:, None]], 1)
        assert all(torch.equal(x, seq) for x in got), kw
    greedy = model.generate(idx, n, top_k=1)
    assert torch.equal(model.generate(idx, n, temperature=0.0, top_p=0.9), greedy)
    assert torch.equal(model.generate(idx, n, top_p=0.0), greedy)
    with pytest.raises(ValueError, match="top_p"):
        model.generate(idx, n, top_p=1.5)


def test_generate_without_them_is_as_before(gpu):
    """temperature and top_k alone: torch's own draw, number for number."""
    cfg = cg.GPTConfig.gpt_nano()
    model = cg.CutileGPT(cfg, dtype=F32, seed=5)
    idx = torch.randint(0, cfg.vocab_size, (2, 6), generator=torch.Generator().manual_seed(1)).to(gpu)
    torch.manual_seed(3)
    got = model.generate(idx, 5, temperature=0.8, top_k=30, use_cache=False)
    torch.manual_seed(3)
    seq = idx
    for _ in range(5):
        x = model(seq)[0][:, -1].float() / 0.8
        x = x.masked_fill(x < torch.topk(x, 30, -1).values[:, -1:], float("-inf"))
        seq = torch.cat([seq, torch.multinomial(torch.softmax(x, -1), 1)], 1)
    assert torch.equal(got, seq)
