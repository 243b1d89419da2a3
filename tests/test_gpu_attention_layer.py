"""The operators together, as a served model runs them: `PagedSelfAttention` as the `self_attn` of the layer
schedules, over a prompt and then single tokens."""
import pytest
import torch

import tokenweave_amd as tw
from kv4_reference import quantise

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H, HQ, HK, D, PAGE, EPS = 512, 4, 1, 64, 16, 1e-5


def attention(cache, seed=3, tp_size=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rotary = tw.RotaryPositions(D, D, 4096, interleaved=False).to(DEV)
    attn = tw.PagedSelfAttention(H, HQ, HK, D, rotary, cache, qkv_bias=True, tp_size=tp_size).to(DEV)
    for p in (attn.qkv_weight, attn.qkv_bias, attn.o_proj.weight):
        p.data.copy_(torch.randn(p.shape, generator=g, device=DEV) * (0.02 if p.dim() == 1 else p.shape[1] ** -0.5))
    return attn


def batch(cache, lengths, news, table):
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    positions = torch.cat([torch.arange(n - m, n) for n, m in zip(lengths, news)]).to(DEV)
    rows = torch.cat([torch.full((m,), i) for i, m in enumerate(news)]).to(DEV)
    slots = table[rows, positions // PAGE].long() * PAGE + positions % PAGE
    return positions, tw.CachedBatch(slots, table, torch.tensor(lengths, dtype=torch.int32, device=DEV),
                                     torch.tensor(starts, dtype=torch.int32, device=DEV), max(news))


def plain(attn, x, seqs):
    """fp32 statement of one call for whole sequences, rounding where the ops do."""
    qkv = (x.float() @ attn.qkv_weight.float().T).bfloat16()
    qkv = (qkv.float() + attn.qkv_bias.float()).bfloat16()
    out, first = [], 0
    for n in seqs:
        q, k, v = (t.view(n, -1, D) for t in qkv[first:first + n].split((HQ * D, HK * D, HK * D), 1))
        first += n
        cos, sin = attn.rotary.cos_sin[:n, None].chunk(2, -1)
        turn = lambda t: torch.cat((t[..., :D // 2] * cos - t[..., D // 2:] * sin,  # noqa: E731
                                    t[..., D // 2:] * cos + t[..., :D // 2] * sin), -1).bfloat16()
        q, k = turn(q.float()), turn(k.float())
        k, v = (quantise(t).float().to(DEV).repeat_interleave(HQ // HK, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q.float(), k) * D ** -0.5
        s = s.masked_fill(torch.ones(n, n, device=DEV).triu(1).bool(), float("-inf"))
        out.append(torch.einsum("hqk,khd->qhd", s.softmax(-1), v).reshape(n, -1).bfloat16())
    return torch.cat(out).float() @ attn.o_proj.weight.float().T


def test_prompt_then_single_tokens_equals_the_whole_sequence():
    """A prompt in one call and the tokens after it one by one attend to the same cache: the last rows are
    those of the whole sequences' plain attention."""
    seqs, prompt = [37, 50], [33, 46]
    cache = tw.KVCache4(9, PAGE, HK, D, DEV)
    cache.pages.fill_(0xFF)
    attn = attention(cache)
    table = torch.tensor([[5, 0, 7, -1], [1, 8, 2, 3]], dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    xs = [torch.randn(n, H, generator=g, device=DEV).bfloat16() for n in seqs]
    got = [[], []]
    x = torch.cat([t[:n] for t, n in zip(xs, prompt)])
    positions, step = batch(cache, prompt, prompt, table)
    attn.begin(step)
    attn(positions=positions, hidden_states=x)
    for i, t in enumerate(x.split(prompt)):
        got[i].append(t)
    for j in range(4):
        lengths = [n + j + 1 for n in prompt]
        x = torch.stack([t[n + j] for t, n in zip(xs, prompt)])
        positions, step = batch(cache, lengths, [1, 1], table)
        attn.begin(step)
        attn(positions=positions, hidden_states=x)
        for i in range(2):
            got[i].append(x[i:i + 1])
    want = plain(attn, torch.cat(xs), seqs)
    torch.testing.assert_close(torch.cat(got[0] + got[1]).float(), want, rtol=1.6e-2, atol=1e-2)


class Layer:
    """A decoder layer whose attention is the package's and whose MLP is a row-parallel projection."""

    def __init__(self, buf, cache, ranks, seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.buf = buf
        self.self_attn = attention(cache, seed, ranks)
        self.input_layernorm, self.post_attention_layernorm = (tw.RMSNorm(H, eps=EPS, dtype=torch.bfloat16).to(DEV)
                                                               for _ in range(2))
        self.down = tw.RowParallelLinear(H, H, bias=False).to(DEV)
        self.down.weight.data.copy_(torch.randn(H, H, generator=g, device=DEV) * H ** -0.5)

    def mlp(self, hidden_states, gemm_cus=None):
        self.down(hidden_states.clone(), hidden_states, is_tokenweave=True, gemm_cus=gemm_cus)


def run_layers(lengths, news, woven):
    """Two layers; the other ranks' partial sums are zero."""
    T, ranks, layers = sum(news), 2, 2
    buf = tw.PartialsBuffer(ranks, T, H, rank=0, device=DEV)
    buf.storage.zero_()
    pages = sum(-(-n // PAGE) for n in lengths)
    table = torch.full((len(lengths), max(-(-n // PAGE) for n in lengths)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(lengths):
        c = -(-n // PAGE)
        table[i, :c] = torch.arange(at, at + c)
        at += c
    g = torch.Generator(device=DEV).manual_seed(9)
    caches = [tw.KVCache4(pages, PAGE, HK, D, DEV) for _ in range(layers)]
    for cache in caches:    # what earlier steps left
        old = torch.randn(pages * PAGE, HK, D, generator=g, device=DEV)
        cache.append(old, old.flip(0), torch.arange(pages * PAGE, device=DEV))
    stack = [Layer(buf, cache, 1, 20 + i) for i, cache in enumerate(caches)]
    positions, step = batch(caches[0], lengths, news, table)
    final = tw.RMSNorm(H, eps=EPS, dtype=torch.bfloat16).to(DEV)
    hidden = buf.hidden_states(T)
    hidden.copy_(torch.randn(T, H, generator=g, device=DEV).bfloat16())
    residual = torch.empty_like(hidden)
    cur, side = torch.cuda.current_stream(), torch.cuda.Stream()
    for i, layer in enumerate(stack):
        layer.self_attn.begin(step)
        nxt = stack[i + 1].input_layernorm if i + 1 < layers else final
        if woven:
            tw.tokenweave_overlap(layer, positions, hidden, residual, buf, i, end_layer=layers, rank=0, world_size=ranks,
                                  current_stream=cur, copy_stream=side, next_layer_norm=nxt,
                                  split_size=tw.tokenweave_split_size(T), actual_tokens=T, num_tokens_padded=T,
                                  MAX_CTAS_ATTN=16, MAX_CTAS_MLP=16, mlp_fn=layer.mlp, all_ranks=True)
        else:
            tw.tokenweave_with_fuse_only(layer, positions, hidden, residual, buf, i, rank=0, world_size=ranks,
                                         next_layer_norm=nxt, actual_tokens=T, nearest_multiple_of_world_size=T,
                                         MAX_CTAS_ATTN=0, MAX_CTAS_MLP=0, mlp_fn=layer.mlp, all_ranks=True)
    torch.cuda.synchronize()
    return hidden.clone(), residual.clone(), [c.pages.clone() for c in caches]


def test_woven_layers_equal_the_unsplit_ones():
    """The schedule's two token splits, a sequence across the boundary among them, see the same cache.  Rows
    are worked on in other groups, so that sums may be taken in another order: 16-bit results differ by
    roundings at most, two layers deep."""
    lengths, news = [300, 150, 77, 400], [200, 150, 1, 289]
    y0, r0, pages0 = run_layers(lengths, news, False)
    y1, r1, pages1 = run_layers(lengths, news, True)
    assert torch.equal(pages0[0], pages1[0])       # the first layer's cache: same inputs, same bits
    torch.testing.assert_close(r1.float(), r0.float(), rtol=1.6e-2, atol=5e-2)
    torch.testing.assert_close(y1.float(), y0.float(), rtol=1.6e-2, atol=5e-2)
    assert float((y1.float() - y0.float()).norm() / y0.float().norm()) < 1e-2


def test_begin_comes_first():
    attn = attention(tw.KVCache4(1, PAGE, HK, D, DEV))
    x = torch.zeros(1, H, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="begin"):
        attn(positions=torch.zeros(1, dtype=torch.int64, device=DEV), hidden_states=x)
