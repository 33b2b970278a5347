"""A decoder layer step by step through a prompt, decode steps, draft rows and another chunk: every stage against its definition, from
the inputs that the stage really got (64-bit formulas for the attention half, the oracle for norms, routing and experts)."""
import numpy as np
import pytest
import torch

from oracle import exl3_oracle as O
from tests import attention_reference as R
from tests.helpers import assert_close_rows
from tests.test_gpu_decode import make

pytestmark = pytest.mark.gpu

HIDDEN, INTER, HEADS, KV_HEADS, DIM, PAGE = 512, 256, 8, 2, 64, 16
# rows and context of three sequences, step by step; the last step leaves one of them out and has rows of nobody behind the others
STEPS = [([37, 5, 20], [37, 5, 20], 0), ([1, 1, 1], [38, 6, 21], 0), ([4, 4, 4], [42, 10, 25], 0), ([30, 0, 2], [72, 10, 27], 3)]


def product_bound(a, b):
    """What a product in FP32 of BF16 operands, rounded once to BF16, may be off: [rows][n] for a [rows][k], b [n][k]."""
    size = a.abs() @ b.abs().T
    return 2.0 ** -8 * (a @ b.T).abs() + a.shape[1] * 2.0 ** -23 * size


@pytest.fixture
def layer(gpu):
    from padra_b200.attention import AttentionKernels, KvCache, Rotary
    from padra_b200.decoder import DecoderLayer, LayerWeights

    g = torch.Generator().manual_seed(3)
    host, _, experts = make(1, HIDDEN, INTER, 4, 91, gpu)
    width = HEADS * DIM

    def matrix(n, k):
        return (torch.randn((n, k), generator=g) * k ** -0.5).bfloat16()

    def norm(n):
        return (1 + 0.2 * torch.randn(n, generator=g)).bfloat16()

    cpu = dict(input_norm=norm(HIDDEN), qkv=matrix(width + 2 * KV_HEADS * DIM, HIDDEN), q_norm=norm(DIM), k_norm=norm(DIM), output=matrix(HIDDEN, width),
               post_norm=norm(HIDDEN), router=matrix(64, HIDDEN))
    inv_freq, amplitude = R.yarn_like(DIM // 2, 4.0)

    class Recorded(AttentionKernels):
        def attention(self, cache, sequences, q, *args, **kwargs):
            self.q = q.clone()
            self.mixed = super().attention(cache, sequences, q, *args, **kwargs)
            return self.mixed

    class Watched(DecoderLayer):
        def attend(self, q, k, v, sequences):
            self.qkv = [t.clone() for t in (q, k, v)]
            self.residual = super().attend(q, k, v, sequences)
            return self.residual

        def feed_forward(self, x, normalized):
            self.middle = x.clone(), normalized.clone()
            super().feed_forward(x, normalized)

    cache = KvCache(24, PAGE, KV_HEADS, DIM, gpu)
    layer = Watched(0, LayerWeights(**{k: v.to(gpu) for k, v in cpu.items()}), Recorded(gpu), experts, cache, Rotary(inv_freq.to(gpu), False, amplitude))
    layer.cpu, layer.host, layer.inv_freq, layer.amplitude, layer.g = cpu, host, inv_freq, amplitude, g
    layer.table = torch.randperm(24, generator=g)[:15].view(3, 5).int()
    return layer


def sequences(layer, rows, context, spare):
    from padra_b200.attention import Sequences

    begin = torch.tensor([0] + rows, dtype=torch.int32).cumsum(0, dtype=torch.int32)
    dev = layer.cache.pool.device
    return Sequences(layer.table.to(dev), begin.to(dev), torch.tensor(context, dtype=torch.int32, device=dev), sum(rows) + spare, max(rows))


def bits(w):
    return w.view(torch.int16).numpy().view(np.uint16)


def check(oracle, layer, x, got, rows, context, pool):
    """`pool`: the cache before the step (CPU), brought up to date here."""
    w, total = layer.cpu, sum(rows)
    # norm + projection
    x0, normalized, _, bad = oracle.residual_norm(x, None, bits(w["input_norm"]))
    assert not bad
    a = torch.from_numpy(normalized).double()
    qkv = torch.cat([t.flatten(1).cpu().double() for t in layer.qkv], 1)
    b = w["qkv"].double()
    assert ((qkv - a @ b.T).abs() <= product_bound(a, b)).all()
    # append and attention, from the projection's bits
    q, k, v = (t.cpu() for t in layer.qkv)
    q_got, mixed = layer.attention.q.cpu().double(), layer.attention.mixed.cpu().double()
    at = 0
    for s, (n, c) in enumerate(zip(rows, context)):
        here, positions = slice(at, at + n), torch.arange(c - n, c)
        keys = R.rotate(R.rms(k[here], w["k_norm"], 1e-6), positions, layer.inv_freq, False, layer.amplitude)
        for r in range(n):
            p = c - n + r
            for h in range(KV_HEADS):
                R.store(pool, int(layer.table[s, p // PAGE]), h, p % PAGE, PAGE, keys[r, h], v[at + r, h].double())
        want = R.rotate(R.rms(q[here], w["q_norm"], 1e-6), positions, layer.inv_freq, False, layer.amplitude)
        slack = 2.0 ** -19 * 2 * layer.amplitude * want.abs().amax(-1, keepdim=True) * 2 ** 0.5 if n else 0
        assert ((q_got[here] - want).abs() <= 2.0 ** -8 * want.abs() + slack).all()
        ks, vs = R.tokens(pool, layer.table[s], c, PAGE, DIM)
        out, bound = R.attention(q_got[here], ks, vs, c - n, DIM ** -0.5, 0)
        assert ((mixed[here] - out).abs() <= bound + 2.0 ** -8 * out.abs() + 1e-7).all()
        at += n
    assert torch.equal(layer.cache.pool.cpu(), pool)
    assert not mixed[total:].any()
    # output projection, residual, second norm
    residual = layer.residual.cpu()
    b = w["output"].double()
    assert ((residual.double() - mixed.flatten(1) @ b.T).abs() <= product_bound(mixed.flatten(1), b)).all()
    x1, normalized, _, bad = oracle.residual_norm(x0, residual.numpy(), bits(w["post_norm"]))
    assert not bad
    assert np.array_equal(layer.middle[0].cpu().numpy(), x1) and np.array_equal(layer.middle[1].cpu().numpy(), normalized)
    # routing and experts, from the router's own product
    logits = (layer.middle[1].bfloat16() @ layer.weights.router.T).float().cpu().numpy()
    ids, routing, bad = oracle.route(logits)
    assert not bad
    _, bad, (_, _, _, down) = oracle.moe_layer(layer.host.table, 0, ids, routing, normalized, HIDDEN, INTER, capture=True)
    want = oracle.combine(x1, down, routing)
    want = want[0] if isinstance(want, tuple) else want
    assert not bad
    assert_close_rows(got, want, "layer output", chained=True)


def test_prompt_decode_drafts_and_another_chunk(oracle, gpu, layer):
    pool = layer.cache.pool.cpu()
    for rows, context, spare in STEPS:
        x = O.bf16_round(torch.randn((sum(rows) + spare, HIDDEN), generator=layer.g).numpy())
        got = layer(torch.from_numpy(x).to(gpu), sequences(layer, rows, context, spare))
        assert layer.attention.bad_flag() == 0 and layer.experts.bad_flag() == 0
        check(oracle, layer, x, got.cpu().numpy(), rows, context, pool)


def test_a_captured_step_is_replayed_with_other_rows(gpu, layer):
    from padra_b200.decoder import DecoderLayer

    plain = DecoderLayer(0, layer.weights, layer.attention, layer.experts, layer.cache, layer.rotary)
    for rows, contexts in (([1, 1, 1], ([40, 3, 80], [41, 4, 17])), ([9, 20, 1], ([40, 20, 80], [9, 33, 1]))):
        seq, x = sequences(layer, rows, contexts[0], 0), torch.zeros((sum(rows), HIDDEN), device=gpu)
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):  # workspaces are made here
            plain(x, seq)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            plain(x, seq)
        for context in contexts:
            seq.context.copy_(torch.tensor(context, dtype=torch.int32))
            fresh = torch.randn(x.shape, generator=layer.g).bfloat16().float().to(gpu)
            pool = layer.cache.pool.clone()
            x.copy_(fresh)
            graph.replay()
            torch.cuda.synchronize()
            got, after = x.clone(), layer.cache.pool.clone()
            layer.cache.pool.copy_(pool)
            want = plain(fresh, seq)
            assert torch.equal(got, want) and torch.equal(after, layer.cache.pool)
    assert layer.attention.bad_flag() == 0 and layer.experts.bad_flag() == 0


def test_refusals(gpu, layer):
    from padra_b200.decoder import DecoderLayer, LayerWeights

    seq = sequences(layer, [1, 1, 1], [5, 5, 5], 0)
    for x in (torch.zeros((2, HIDDEN), device=gpu), torch.zeros((3, HIDDEN), device=gpu, dtype=torch.bfloat16), torch.zeros((3, HIDDEN // 2), device=gpu)):
        with pytest.raises(ValueError):
            layer(x, seq)
    w = dict(vars(layer.weights))
    for name, value in (("qkv", w["qkv"][:-DIM]), ("output", w["output"][:, :-8]), ("router", w["router"][:63]), ("post_norm", w["post_norm"].float())):
        with pytest.raises(ValueError):
            DecoderLayer(0, LayerWeights(**{**w, name: value}), layer.attention, layer.experts, layer.cache)
    empty = torch.zeros((0, HIDDEN), device=gpu)
    assert layer(empty, sequences(layer, [0, 0, 0], [5, 5, 5], 0)) is empty


@pytest.mark.parametrize("rows", [17, 2050])
def test_chunks_longer_than_one_schedule(gpu, layer, rows):
    """2050 rows are a chunk of 2048 and a tail of two: every part as if it were alone."""
    g = torch.Generator().manual_seed(rows)
    normalized = torch.randn((rows, HIDDEN), generator=g).bfloat16().float().to(gpu)
    x = torch.randn((rows, HIDDEN), generator=g).bfloat16().float().to(gpu)
    got = x.clone()
    layer.feed_forward(got, normalized)
    logits = (normalized.bfloat16() @ layer.weights.router.T).float()
    for at in range(0, rows, 2048):
        n = min(2048, rows - at)
        want, part = x[at:at + n].clone(), slice(at, at + n)
        ids, routing = layer.experts.route(logits[part])
        if n > 3:
            layer.experts.prefill_layer(0, ids.reshape(-1), routing.reshape(-1), normalized[part].contiguous(), want, n)
        else:
            layer.experts.moe_decode_layer(0, ids, routing, normalized[part].contiguous(), want, n)
        assert torch.equal(got[part], want)
    assert layer.experts.bad_flag() == 0 and not torch.equal(got, x)
