"""Per-head norm and rotation, the paged 4-bit cache and attention over it, against the formulas in 64 bits
(tests/attention_reference.py).  The refusals run on the CPU: they come from the C ABI's argument checks."""
import ctypes as C
import math
import threading
import time

import pytest
import torch

from tests import attention_reference as R

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative


# ---- refusals (CPU) -------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def lib():
    from padra_b200 import binding, build

    build.build()
    return binding.load()


def structs(**over):
    """Plausible structs over addresses that are never read."""
    from padra_b200 import binding as B

    c = dict(pool=4096, pages=4, page_size=16, kv_heads=2, head_dim=64)
    s = dict(page_table=4096, row_begin=4096, context=4096, count=1, table_stride=2, rows=3, max_rows=3)
    r = dict(inv_freq=4096, amplitude=1.0, dims=64, interleaved=0)
    for k, v in over.items():
        for d in (c, s, r):
            if k in d:
                d[k] = v
    return B.KvCacheStruct(**c), B.SequencesStruct(**s), B.RotaryStruct(**r)


@pytest.mark.parametrize("over, status", [
    (dict(pool=4100), "INVALID_ARGUMENT"), (dict(pool=None), "INVALID_ARGUMENT"), (dict(pages=0), "INVALID_ARGUMENT"), (dict(pages=1 << 31), "INVALID_ARGUMENT"),
    (dict(page_size=8), "INVALID_ARGUMENT"), (dict(page_size=48), "INVALID_ARGUMENT"), (dict(page_size=512), "INVALID_ARGUMENT"), (dict(kv_heads=0), "INVALID_ARGUMENT"),
    (dict(head_dim=96), "UNSUPPORTED"), (dict(head_dim=256), "UNSUPPORTED"), (dict(count=-1), "INVALID_ARGUMENT"), (dict(rows=-1), "INVALID_ARGUMENT"),
    (dict(table_stride=1 << 27), "INVALID_ARGUMENT"), (dict(row_begin=None), "INVALID_ARGUMENT"), (dict(page_table=None), "INVALID_ARGUMENT")])
def test_cache_and_sequences_are_checked_before_anything_is_enqueued(lib, over, status):
    from padra_b200 import binding as B

    c, s, r = structs(**over)
    want = getattr(B, status)
    p = 4096
    assert lib.padra_kv_append(C.byref(c), C.byref(s), p, p, 256, 256, None, 1e-6, None, None, None, 0, 0, 0, None, 0, p, None) == want
    assert lib.padra_kv_read(C.byref(c), C.byref(s), p, p, 256, 256, 0, p, None) == want
    assert lib.padra_attention_q4(C.byref(c), C.byref(s), p, p, 512, 512, 4, 0, 0.1, 0, p, 1 << 40, p, None) == want


def test_row_arguments_are_checked(lib):
    from padra_b200 import binding as B

    c, s, r = structs()
    p = 4096
    ok = [C.byref(c), C.byref(s), p, p, 512, 512, 4, 0, 0.1, 0, p, lib.padra_attention_q4_workspace_bytes(64), p, None]
    for at, value, want in [(2, p + 2, B.INVALID_ARGUMENT), (2, None, B.INVALID_ARGUMENT), (3, p + 8, B.INVALID_ARGUMENT), (4, 255, B.INVALID_ARGUMENT),
                            (4, 260, B.INVALID_ARGUMENT), (5, 128, B.INVALID_ARGUMENT), (6, 3, B.INVALID_ARGUMENT), (6, 0, B.INVALID_ARGUMENT),
                            (7, B.ROWS_F32, B.UNSUPPORTED), (7, 9, B.UNSUPPORTED), (8, math.inf, B.INVALID_ARGUMENT), (9, -1, B.INVALID_ARGUMENT), (10, None, B.INVALID_ARGUMENT),
                            (10, p + 8, B.INVALID_ARGUMENT), (11, lib.padra_attention_q4_workspace_bytes(64) - 1, B.INVALID_ARGUMENT), (12, None, B.INVALID_ARGUMENT)]:
        args = list(ok)
        args[at] = value
        assert lib.padra_attention_q4(*args) == want, (at, value)
    rope = [p, p, 256, 256, 4, None, None, 0, 0, 0, None, None, 1e-6, p, C.byref(r), 3, 64, 0, p, None]
    for at, value, want in [(0, p + 4, B.INVALID_ARGUMENT), (2, 200, B.INVALID_ARGUMENT), (4, 0, B.INVALID_ARGUMENT), (9, 1, B.INVALID_ARGUMENT), (10, p + 2, B.INVALID_ARGUMENT),
                            (12, -1.0, B.INVALID_ARGUMENT), (12, math.nan, B.INVALID_ARGUMENT), (13, None, B.INVALID_ARGUMENT), (16, 80, B.UNSUPPORTED), (17, 3, B.UNSUPPORTED), (18, None, B.INVALID_ARGUMENT)]:
        args = list(rope)
        args[at] = value
        assert lib.padra_qk_norm_rope(*args) == want, (at, value)
    for dims in (8, 24, 80, 128, -16):
        _, _, bad = structs(dims=dims)
        args = list(rope)
        args[14] = C.byref(bad)
        assert lib.padra_qk_norm_rope(*args) == B.INVALID_ARGUMENT, dims
    append = [C.byref(c), C.byref(s), p, p, 128, 128, None, 1e-6, C.byref(r), p, p, 256, 256, 4, None, 0, p, None]
    for at, value, want in [(2, p + 4, B.INVALID_ARGUMENT), (5, 120, B.INVALID_ARGUMENT), (10, None, B.INVALID_ARGUMENT), (13, 0, B.INVALID_ARGUMENT), (15, 5, B.UNSUPPORTED)]:
        args = list(append)
        args[at] = value
        assert lib.padra_kv_append(*args) == want, (at, value)


def test_attention_workspace(lib):
    assert lib.padra_attention_q4_workspace_bytes(96) == 0
    assert 0 < lib.padra_attention_q4_workspace_bytes(64) < lib.padra_attention_q4_workspace_bytes(128)


def test_nothing_to_do_is_not_an_error(lib):
    from padra_b200 import binding as B

    p = 4096
    for over in (dict(rows=0), dict(count=0, row_begin=None, context=None)):
        c, s, r = structs(**over)
        assert lib.padra_attention_q4(C.byref(c), C.byref(s), p, p, 512, 512, 4, 0, 0.1, 0, p, 1 << 40, p, None) == B.OK
        assert lib.padra_kv_read(C.byref(c), C.byref(s), p, p, 128, 128, 0, p, None) == B.OK
        assert lib.padra_kv_append(C.byref(c), C.byref(s), p, p, 128, 128, None, 1e-6, None, None, None, 0, 0, 0, None, 0, p, None) == B.OK
    assert lib.padra_qk_norm_rope(p, p, 256, 256, 4, None, None, 0, 0, 0, None, None, 1e-6, p, None, 0, 64, 0, p, None) == B.OK


def test_row_arrays_without_rows_need_no_memory(lib):
    """As a framework's empty tensors, whose address is null."""
    from padra_b200 import binding as B

    p = 4096
    c, s, r = structs(rows=0)
    assert lib.padra_attention_q4(C.byref(c), C.byref(s), None, None, 512, 512, 4, 0, 0.1, 0, p, 1 << 40, p, None) == B.OK
    assert lib.padra_kv_read(C.byref(c), C.byref(s), None, None, 128, 128, 0, p, None) == B.OK
    assert lib.padra_kv_append(C.byref(c), C.byref(s), None, None, 128, 128, None, 1e-6, C.byref(r), None, None, 256, 256, 4, None, 0, p, None) == B.OK
    assert lib.padra_qk_norm_rope(None, None, 256, 256, 4, None, None, 128, 128, 2, None, None, 1e-6, None, C.byref(r), 0, 64, 0, p, None) == B.OK
    # what is wrong in itself is refused all the same
    assert lib.padra_attention_q4(C.byref(c), C.byref(s), None, None, 255, 512, 4, 0, 0.1, 0, p, 1 << 40, p, None) == B.INVALID_ARGUMENT
    assert lib.padra_attention_q4(C.byref(c), C.byref(s), None, None, 512, 512, 4, B.ROWS_F32, 0.1, 0, p, 1 << 40, p, None) == B.UNSUPPORTED
    assert lib.padra_kv_read(C.byref(c), C.byref(s), None, None, 120, 128, 0, p, None) == B.INVALID_ARGUMENT
    assert lib.padra_qk_norm_rope(p + 4, None, 256, 256, 4, None, None, 0, 0, 0, None, None, 1e-6, None, None, 0, 64, 0, p, None) == B.INVALID_ARGUMENT


def test_python_side_checks_shapes_and_types():
    from padra_b200 import attention as A

    with pytest.raises(ValueError):
        A.KvCache(2, 16, 1, 96, device="cpu")
    with pytest.raises(ValueError):
        A.KvCache.over(torch.zeros((2, 1, 100), dtype=torch.uint8), 16, 64)
    with pytest.raises(ValueError):
        A.Rotary(torch.zeros(32))
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        A.Sequences(i[None], i, i, 4, 4)
    with pytest.raises(ValueError):
        A.Sequences(torch.zeros((3, 1), dtype=torch.int64), torch.zeros(4, dtype=torch.int32), i, 4, 4)


def test_first_calls_of_two_threads_get_one_workspace(monkeypatch):
    from types import SimpleNamespace

    from padra_b200 import attention as A

    def slowly(head_dim):
        time.sleep(0.05)
        return 4096

    k = A.AttentionKernels.__new__(A.AttentionKernels)  # without a device
    k.lib, k.bad, k._workspace, k._making = SimpleNamespace(padra_attention_q4_workspace_bytes=slowly), torch.zeros(1), {}, threading.Lock()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    got = []
    threads = [threading.Thread(target=lambda: got.append(k.workspace(64, 0))) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 4 and set(got) == {(k._workspace[0, 64][0], 4096)}


def test_reference_quantiser_against_a_plain_loop():
    g = torch.Generator().manual_seed(3)
    x = torch.randn((2, 64), generator=g, dtype=torch.float64)
    x[1, 32:] = 0
    codes, scales = R.quantise(x)
    for r in range(2):
        for b in range(2):
            most = max(abs(float(t)) for t in x[r, 32 * b:32 * b + 32])
            s = float(torch.tensor(most / 7, dtype=torch.float64).to(torch.float16))
            assert abs(float(scales[r, b]) - s) <= s * 2 ** -10
            for d in range(32):
                t = float(x[r, 32 * b + d])
                assert int(codes[r, 32 * b + d]) == (round(t / float(scales[r, b])) + 8 if s else 8)
    pool = torch.zeros((1, 1, 16 * 72), dtype=torch.uint8)
    R.store(pool, 0, 0, 5, 16, x[0], x[1])
    k, v = R.fetch(pool, 0, 16, 64)
    assert torch.equal(k[0, 5], R.dequantise(codes, scales)[0]) and torch.equal(v[0, 5], R.dequantise(codes, scales)[1])


MARKED = [(8, 2, 1, 40000), (16, 1, 1, 40000), (24, 1, 1, 20000), (8, 2, 2, 9001), (8, 1, 5, 9001), (12, 1, 4, 16001), (300, 1, 1, 5000), (16, 1, 33, 4100), (8, 2, 300, 2500),
          (4, 1, 130, 6000), (8, 1, 200, 20011)]


def marked_bound(want, dtype):
    """One rounding of the output; sums of exact terms in 32 bits are far below the rest (2^-14: 2^10 additions in a row of half a step of
    2^-23 each, should an addition truncate)."""
    return HALF[dtype] * want + 2.0 ** -14 * want


@pytest.mark.parametrize("heads, kv_heads, rows, context", MARKED)
def test_the_bound_of_marked_sequences_shows_every_lost_or_doubled_tile(heads, kv_heads, rows, context):
    k, v, want = R.marked(rows, context, 64)
    last = min(rows, 3)  # rows at the end see every tile
    weight = 2.0 ** k[:, 0]
    for tile in range((context - rows) // 32):  # whole tiles that every row sees
        here = slice(32 * tile, 32 * tile + 32)
        part, share = weight[here] @ v[here], weight[here].sum()
        for r in range(rows - last, rows):
            total = weight[:context - rows + r + 1].sum()
            for times in (-1, 1):
                got = (want[r] * total + times * part) / (total + times * share)
                assert ((got - want[r]).abs() > 2 * marked_bound(want[r], torch.bfloat16)).any(), tile


# ---- GPU ----------------------------------------------------------------------------------------------------------------

class Call:
    """A pool, a page table in random order and rows for ragged sequences, on both sides."""

    def __init__(self, gpu, shapes, heads, kv_heads, dim, page, dtype, seed, spare_rows=0, spare_pages=2, strided=True):
        from padra_b200 import attention as A

        g = self.g = torch.Generator().manual_seed(seed)
        self.shapes, self.heads, self.kv_heads, self.dim, self.page, self.dtype, self.gpu = shapes, heads, kv_heads, dim, page, dtype, gpu
        need = [-(-c // page) for _, c in shapes]
        pages = sum(need) + spare_pages
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((len(shapes), max(need + [1])), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.begin = torch.tensor([0] + [n for n, _ in shapes], dtype=torch.int32).cumsum(0, dtype=torch.int32)
        self.context = torch.tensor([c for _, c in shapes], dtype=torch.int32)
        self.rows = int(self.begin[-1]) + spare_rows
        # anything a former user may have left in the pages, with finite scales
        self.pool = torch.randint(0, 256, (pages, kv_heads, A.KvCache.block_bytes(page, dim)), generator=g, dtype=torch.uint8)
        a, b = page * dim // 2, page * dim // 16
        for at in (a, 2 * a + b):
            n = pages * kv_heads * page * dim // 32
            self.pool[:, :, at:at + b] = (torch.rand(n, generator=g) * 0.4).to(torch.float16).view(torch.uint8).view(pages, kv_heads, b)
        width = (heads + 2 * kv_heads) * dim + (16 if strided else 0)
        self.qkv = torch.randn((self.rows, width), generator=g).to(dtype)
        self.split()
        self.kernels = A.AttentionKernels(gpu)
        self.cache = A.KvCache.over(self.pool.to(gpu), page, dim)
        self.d_qkv = self.qkv.to(gpu)
        self.dq, self.dk, self.dv = self.views(self.d_qkv)
        self.sequences = A.Sequences(self.table.to(gpu), self.begin.to(gpu), self.context.to(gpu), self.rows, max([n for n, _ in shapes] + [0]))

    def views(self, qkv):
        h, kv, d = self.heads, self.kv_heads, self.dim
        return (qkv[:, :h * d].unflatten(1, (h, d)), qkv[:, h * d:(h + kv) * d].unflatten(1, (kv, d)), qkv[:, (h + kv) * d:(h + 2 * kv) * d].unflatten(1, (kv, d)))

    def split(self):
        self.q, self.k, self.v = self.views(self.qkv)

    def reference(self, scale, window, pool=None):
        pool = self.pool if pool is None else pool
        want, bound = torch.zeros((self.rows, self.heads, self.dim), dtype=torch.float64), torch.zeros((self.rows, self.heads, self.dim), dtype=torch.float64)
        for s, (n, c) in enumerate(self.shapes):
            b = int(self.begin[s])
            k, v = R.tokens(pool, self.table[s], c, self.page, self.dim)
            want[b:b + n], bound[b:b + n] = R.attention(self.q[b:b + n], k, v, c - n, scale, window)
        return want, bound

    def check_attention(self, scale=None, window=0, what="attention"):
        scale = self.dim ** -0.5 if scale is None else scale
        out = torch.full((self.rows, self.heads, self.dim), 7.0, dtype=self.dtype, device=self.gpu)
        self.kernels.attention(self.cache, self.sequences, self.dq, scale, window, out)
        assert self.kernels.bad_flag() == 0
        got, last = out.cpu().double(), int(self.begin[-1])
        want, bound = self.reference(scale, window)
        assert (got[last:] == 7).all(), "rows behind the last sequence were touched"
        off = (got[:last] - want[:last]).abs() - (bound[:last] + HALF[self.dtype] * want[:last].abs() + 1e-7)
        assert off.max().item() <= 0 if off.numel() else True, f"{what}: {off.max().item():.3e} beyond the bound"
        return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows, heads, kv_heads, dim, dims, interleaved, norm", [
    (1, 1, 1, 64, 64, False, True), (1, 32, 4, 128, 128, False, True), (3, 5, 3, 64, 32, True, True), (7, 7, 1, 128, 64, False, False),
    (601, 4, 2, 64, 16, True, True), (1203, 3, 1, 256, 256, False, True), (33, 2, 2, 256, 48, True, False), (5, 4, 0, 128, 0, False, True)])
def test_norm_and_rotation(gpu, dtype, rows, heads, kv_heads, dim, dims, interleaved, norm):
    from padra_b200 import attention as A

    g = torch.Generator().manual_seed(rows + dim)
    qkv = (torch.randn((rows, heads + kv_heads + 1, dim), generator=g) * torch.exp(torch.randn((rows, 1, 1), generator=g))).to(dtype)
    q, k = qkv[:, :heads], qkv[:, heads:heads + kv_heads] if kv_heads else None
    weights = [(1 + 0.3 * torch.randn(dim, generator=g)).bfloat16() if norm else None for _ in range(2)]
    positions = torch.randint(0, 1 << 17, (rows,), generator=g, dtype=torch.int32)
    positions[0] = 0
    inv_freq, amplitude = R.yarn_like(dims // 2, 4.0) if dims else (torch.zeros(0, dtype=torch.float64), 1.0)
    kernels = A.AttentionKernels(gpu)
    rotary = A.Rotary(inv_freq.to(gpu), interleaved, amplitude) if dims else None
    d = qkv.to(gpu)
    got = kernels.qk_norm_rope(d[:, :heads], d[:, heads:heads + kv_heads] if kv_heads else None, positions.to(gpu), rotary,
                               *[None if w is None else w.to(gpu) for w in weights], 1e-6)
    assert kernels.bad_flag() == 0
    for x, w, y in zip((q, k), weights, got):
        if x is None:
            continue
        normed = R.rms(x, w, 1e-6)
        want = R.rotate(normed, positions, inv_freq, interleaved, amplitude)
        # FP32 on the way: the norm's factor is off by about 14 * 2^-24, products, the reduced angle (2^-22) and sincos (2^-23) add
        # up to less than 2^-19 of the pair's two values
        slack = 2.0 ** -19 * 2 * amplitude * normed.abs().amax(-1, keepdim=True)
        assert ((y.cpu().double() - want).abs() <= HALF[dtype] * want.abs() + slack).all()
    # in place, and the same bits
    kernels.qk_norm_rope(d[:, :heads], d[:, heads:heads + kv_heads] if kv_heads else None, positions.to(gpu), rotary,
                         *[None if w is None else w.to(gpu) for w in weights], 1e-6, d[:, :heads], d[:, heads:heads + kv_heads] if kv_heads else None)
    assert torch.equal(d[:, :heads], got[0]) and (not kv_heads or torch.equal(d[:, heads:heads + kv_heads], got[1]))
    assert torch.equal(d[:, -1].cpu(), qkv[:, -1])


@pytest.mark.gpu
def test_norm_and_rotation_report_what_is_not_finite(gpu):
    from padra_b200 import attention as A

    kernels = A.AttentionKernels(gpu)
    x = torch.ones((2, 1, 64), dtype=torch.float16, device=gpu)
    kernels.qk_norm_rope(x, None, None)
    assert kernels.bad_flag() == 0
    x[1, 0, 3] = float("inf")
    kernels.qk_norm_rope(x, None, None)
    assert kernels.bad_flag() == 1


SHAPES = {
    "one": [(1, 1)], "decode": [(1, 130), (1, 1), (1, 64), (1, 17)], "verify": [(5, 40), (2, 2), (16, 333)],
    "empty": [(0, 0), (1, 33), (0, 20), (3, 3), (0, 0)], "padded": [(4, 2), (1, 0), (3, 3)], "chunk": [(70, 200), (129, 129), (1, 300)]}


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("dtype, heads, kv_heads, dim, page, dims, interleaved, norm", [
    (torch.bfloat16, 8, 2, 128, 64, 128, False, True), (torch.float16, 3, 3, 64, 16, 32, True, True), (torch.float32, 4, 1, 64, 128, 64, False, False),
    (torch.bfloat16, 5, 5, 128, 32, 0, False, True)])
def test_append_writes_the_bytes_of_the_definition(gpu, shapes, dtype, heads, kv_heads, dim, page, dims, interleaved, norm):
    from padra_b200 import attention as A

    c = Call(gpu, SHAPES[shapes], heads, kv_heads, dim, page, dtype, 11, spare_rows=3)
    c.v[0, 0, :32] = 0  # a group of zeros
    if dtype != torch.float16:
        c.v[0, 0, 32:64] = torch.tensor([3.5, -2.5, 1.5, 0.5, 7.0, -7.0, 6.5, 5.5] * 4).to(dtype)  # scale 1: values on the borders
    c.d_qkv.copy_(c.qkv)
    weights = [(1 + 0.3 * torch.randn(dim, generator=c.g)).bfloat16() if norm else None for _ in range(2)]
    inv_freq, amplitude = R.yarn_like(dims // 2, 2.0) if dims else (torch.zeros(0, dtype=torch.float64), 1.0)
    rotary = A.Rotary(inv_freq.to(gpu), interleaved, amplitude) if dims else None
    dw = [None if w is None else w.to(gpu) for w in weights]
    q_out = torch.full((c.rows, heads, dim), 7.0, dtype=dtype, device=gpu)
    c.kernels.append(c.cache, c.sequences, c.dk, c.dv, rotary, dw[1], 1e-6, c.dq, dw[0], q_out)
    assert c.kernels.bad_flag() == 0
    want = c.pool.clone()
    q_want, q_there = torch.full((c.rows, heads, dim), 7.0, dtype=torch.float64), torch.zeros(c.rows, dtype=torch.bool)
    for s, (n, ctx) in enumerate(c.shapes):
        b = int(c.begin[s])
        at = torch.arange(ctx - n, ctx)
        k = R.rotate(R.rms(c.k[b:b + n], weights[1], 1e-6), at, inv_freq, interleaved, amplitude)
        q_want[b:b + n] = R.rotate(R.rms(c.q[b:b + n], weights[0], 1e-6), at, inv_freq, interleaved, amplitude)
        for r in range(n):
            p = ctx - n + r
            q_there[b + r] = p >= 0
            for h in range(kv_heads if p >= 0 else 0):
                R.store(want, int(c.table[s, p // page]), h, p % page, page, k[r, h], c.v[b + r, h].double())
    assert torch.equal(c.cache.pool.cpu(), want)
    got = q_out.cpu().double()
    assert (got[~q_there] == 7).all()
    slack = 2.0 ** -19 * 2 * amplitude * q_want.abs().amax(-1, keepdim=True) * math.sqrt(2)
    assert ((got - q_want).abs() <= HALF[dtype] * q_want.abs() + slack)[q_there].all()
    # and back
    k_back, v_back = (torch.full((c.rows, kv_heads, dim), 7.0, dtype=torch.float32, device=gpu) for _ in range(2))
    c.kernels.read(c.cache, c.sequences, k_back, v_back)
    assert (k_back.cpu()[~q_there] == 7).all()
    for s, (n, ctx) in enumerate(c.shapes):
        k, v = R.tokens(want, c.table[s], ctx, page, dim)
        b, skip = int(c.begin[s]), max(0, n - ctx)
        assert torch.equal(k_back.cpu()[b + skip:b + n].double(), k[ctx - n + skip:]) and torch.equal(v_back.cpu()[b + skip:b + n].double(), v[ctx - n + skip:])
    k16, v16 = c.kernels.read(c.cache, c.sequences, dtype=torch.bfloat16)
    assert torch.equal(k16[q_there], k_back[q_there].bfloat16()) and torch.equal(v16[q_there], v_back[q_there].bfloat16())
    assert c.kernels.bad_flag() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf"), 60000.0])
@pytest.mark.parametrize("which", ["k", "v"])
def test_append_leaves_out_a_head_that_four_bits_cannot_hold(gpu, value, which):
    c = Call(gpu, [(2, 5), (1, 9)], 4, 2, 64, 16, torch.float32, 5)
    getattr(c, which)[1, 1, 40] = value
    c.d_qkv.copy_(c.qkv)
    c.kernels.append(c.cache, c.sequences, c.dk, c.dv)
    assert c.kernels.bad_flag() == 1
    want = c.pool.clone()
    for s, (n, ctx) in enumerate(c.shapes):
        for r in range(n):
            b, p = int(c.begin[s]) + r, ctx - n + r
            for h in range(2):
                page, slot = int(c.table[s, p // 16]), p % 16
                before = R.fetch(want, page, 16, 64)
                k, v = c.k[b, h].double(), c.v[b, h].double()
                if (b, h) == (1, 1):
                    k, v = (before[0][h, slot], v) if which == "k" else (k, before[1][h, slot])
                R.store(want, page, h, slot, 16, k, v)
    got, held = c.cache.pool.cpu(), c.pool
    page, slot = int(c.table[0, 0]), 4
    at = {"k": 0, "v": 16 * 36}[which] + slot * 32  # the head that was refused keeps its bytes
    want[page, 1, at:at + 32] = held[page, 1, at:at + 32]
    at = {"k": 0, "v": 16 * 36}[which] + 16 * 32 + slot * 4
    want[page, 1, at:at + 4] = held[page, 1, at:at + 4]
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads, kv_heads, dim, page", [(8, 2, 128, 64), (3, 3, 64, 16), (7, 1, 128, 16), (8, 1, 64, 128), (6, 2, 128, 256)])
@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("window", [0, 1, 50])
def test_attention(gpu, dtype, heads, kv_heads, dim, page, shapes, window):
    Call(gpu, SHAPES[shapes], heads, kv_heads, dim, page, dtype, 21, spare_rows=2).check_attention(window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_attention_with_other_scales(gpu, scale):
    Call(gpu, [(1, 700), (3, 129), (40, 90)], 8, 2, 128, 64, torch.bfloat16, 23).check_attention(scale=scale)


@pytest.mark.gpu
def test_pages_that_do_not_exist_are_reported_and_not_read(gpu):
    for page in (-1, 10 ** 6):
        c = Call(gpu, [(1, 200), (40, 60), (1, 5)], 4, 2, 64, 16, torch.bfloat16, 31)
        c.sequences.page_table[0, 3] = page
        c.sequences.page_table[1, 1] = page
        c.kernels.attention(c.cache, c.sequences, c.dq, 0.125)
        assert c.kernels.bad_flag() == 1
        c.kernels.reset_bad()
        c.sequences.page_table[0, 12] = page  # the page that the last token goes to
        c.kernels.append(c.cache, c.sequences, c.dk, c.dv)
        assert c.kernels.bad_flag() == 1
        c.kernels.reset_bad()
        c.kernels.read(c.cache, c.sequences)
        assert c.kernels.bad_flag() == 1


@pytest.mark.gpu
@pytest.mark.parametrize("fault", ["context beyond the table", "negative context", "rows beyond the array", "descending rows", "more rows than announced"])
def test_contradicting_sequences_are_reported(gpu, fault):
    c = Call(gpu, [(2, 40), (3, 60)], 4, 2, 64, 16, torch.bfloat16, 33)
    s = c.sequences
    if fault == "context beyond the table":
        s.context[0] = 16 * s.page_table.shape[1] + 1
    elif fault == "negative context":
        s.context[1] = -5
    elif fault == "rows beyond the array":
        s.row_begin[2] = 60
    elif fault == "descending rows":
        s.row_begin[1] = -3
    else:
        s.struct.max_rows = 1
    for call in (lambda: c.kernels.attention(c.cache, s, c.dq, 0.125), lambda: c.kernels.append(c.cache, s, c.dk, c.dv), lambda: c.kernels.read(c.cache, s)):
        call()
        assert c.kernels.bad_flag() == 1
        c.kernels.reset_bad()


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(1, 300), (1, 40)], [(40, 300), (1, 40)]])
def test_queries_that_are_not_finite_are_reported_and_give_zeros(gpu, shapes):
    c = Call(gpu, shapes, 4, 2, 64, 16, torch.bfloat16, 35)
    good = c.check_attention()
    c.dq[0, 1, 5] = float("nan")
    c.dq[shapes[0][0], 3, 0] = float("-inf")
    out = c.kernels.attention(c.cache, c.sequences, c.dq, 64 ** -0.5)
    assert c.kernels.bad_flag() == 1
    hurt = torch.zeros(out.shape[:2], dtype=torch.bool, device=gpu)
    hurt[0, 1] = hurt[shapes[0][0], 3] = True
    assert (out[hurt] == 0).all() and torch.equal(out[~hurt], good[~hurt])


@pytest.mark.gpu
def test_a_pool_of_more_than_four_gigabytes(gpu):
    from padra_b200 import attention as A

    c = Call(gpu, [(1, 200), (20, 90)], 8, 4, 128, 64, torch.bfloat16, 37)
    pages = (5 << 30) // c.pool[0].numel()
    pool = torch.empty((pages,) + c.pool.shape[1:], dtype=torch.uint8, device=gpu)
    shift = pages - c.pool.shape[0]
    pool[shift:] = c.pool.to(gpu)
    pool[:c.pool.shape[0]] = 0
    c.cache = A.KvCache.over(pool, 64, 128)
    c.sequences.page_table += torch.where(c.sequences.page_table >= 0, shift, 0).int()
    c.check_attention()
    c.kernels.append(c.cache, c.sequences, c.dk, c.dv)
    back, _ = c.kernels.read(c.cache, c.sequences, dtype=torch.float32)
    want = R.dequantise(*R.quantise(c.k.double()))
    assert torch.equal(back.cpu().double(), want)
    assert not pool[:c.pool.shape[0]].any() and c.kernels.bad_flag() == 0


def unwritten(c, window):
    """Gives every slot that no row attends to scales that are NaN or infinite (all of K's and V's), on both sides."""
    a, b = c.page * c.dim // 2, c.page * c.dim // 16
    seen = torch.zeros((c.pool.shape[0], c.page), dtype=torch.bool)
    for s, (n, ctx) in enumerate(c.shapes):
        for t in range(max(0, ctx - n - window + 1) if window else 0, ctx if n else 0):
            seen[int(c.table[s, t // c.page]), t % c.page] = True
    for at in (a, 2 * a + b):
        scales = c.pool[:, :, at:at + b].contiguous().view(torch.float16).view(c.pool.shape[0], c.kv_heads, c.page, c.dim // 32)
        scales[~seen[:, None, :].expand(-1, c.kv_heads, -1)] = torch.tensor([float("nan"), float("inf")] * (c.dim // 64), dtype=torch.float16)
        c.pool[:, :, at:at + b] = scales.view(torch.uint8).view(c.pool.shape[0], c.kv_heads, b)
    c.cache.pool.copy_(c.pool)


@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv_heads, dim, page", [(8, 2, 128, 64), (12, 1, 64, 16), (4, 4, 128, 256)])
@pytest.mark.parametrize("shapes", [[(1, 200), (1, 1), (1, 77)], [(3, 150), (2, 19)], [(70, 200), (5, 131), (130, 130)], [(0, 90), (1, 0), (2, 1)]])
@pytest.mark.parametrize("window", [0, 1, 20])
def test_slots_that_nobody_attends_to_may_hold_anything(gpu, heads, kv_heads, dim, page, shapes, window):
    c = Call(gpu, shapes, heads, kv_heads, dim, page, torch.bfloat16, 41, spare_rows=1)
    unwritten(c, window)
    live = c.reference

    def reference(scale, window, pool=None):  # 0 * NaN stays out of the reference too
        held = c.pool
        c.pool = held.clone()
        a, b = c.page * c.dim // 2, c.page * c.dim // 16
        for at in (a, 2 * a + b):
            s = c.pool[:, :, at:at + b].contiguous().view(torch.float16)
            c.pool[:, :, at:at + b] = s.nan_to_num(0, 0, 0).view(torch.uint8)
        try:
            return live(scale, window)
        finally:
            c.pool = held

    c.reference = reference
    c.check_attention(window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv_heads, rows, context", [
    (8, 8, 1, 40000), (8, 2, 1, 40000), (16, 1, 1, 40000), (24, 1, 1, 20000), (300, 1, 1, 5000), (300, 1, 7, 600), (8, 2, 2, 9001), (8, 1, 5, 9001),
    (8, 8, 9, 5000), (16, 1, 33, 2100), (8, 2, 300, 2500), (4, 1, 130, 6000)])
def test_one_sequence_split_over_the_gpu(gpu, heads, kv_heads, rows, context):
    """Many pieces of one unit: few and many joins, one, several and many blocks of columns."""
    Call(gpu, [(rows, context)], heads, kv_heads, 64, 64, torch.bfloat16, 43).check_attention(window=0)


@pytest.mark.gpu
@pytest.mark.parametrize("count, most_rows", [(1, 1), (33, 2), (129, 1), (700, 1), (700, 5), (150, 40)])
def test_many_sequences(gpu, count, most_rows):
    g = torch.Generator().manual_seed(count)
    shapes = []
    for _ in range(count):
        n = int(torch.randint(0, most_rows + 1, (1,), generator=g))
        shapes.append((n, n + int(torch.randint(0, 90, (1,), generator=g))))
    c = Call(gpu, shapes, 4, 2, 64, 16, torch.bfloat16, 47, spare_rows=3)
    c.check_attention()
    c.check_attention(window=9)
    q = c.kernels.append(c.cache, c.sequences, c.dk, c.dv, q=c.dq, q_out=torch.zeros_like(c.dq))
    k, v = c.kernels.read(c.cache, c.sequences, torch.zeros_like(c.dk, dtype=torch.float32), torch.zeros_like(c.dv, dtype=torch.float32))
    last = int(c.begin[-1])
    for x, got in ((c.k, k), (c.v, v)):
        assert torch.equal(got[:last].cpu().double(), R.dequantise(*R.quantise(x[:last].double())))
    assert torch.equal(q[:last], c.dq[:last]) and not q[last:].any() and not k[last:].any() and c.kernels.bad_flag() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 20, 130])
@pytest.mark.parametrize("order", [1, -1])
def test_scores_that_rise_and_fall_along_the_axis(gpu, rows, order):
    """Scores from -100 to 100: the running maximum moves with every tile, or never after the first."""
    c = Call(gpu, [(rows, 1500)], 4, 2, 64, 32, torch.float16, 53)
    c.q[:] = 0.25
    c.d_qkv.copy_(c.qkv)
    for t in range(1500):
        k = torch.full((64,), order * (t - 750) / 750, dtype=torch.float64)
        for h in range(2):
            R.store(c.pool, int(c.table[0, t // 32]), h, t % 32, 32, k, torch.full((64,), float(t % 50), dtype=torch.float64))
    c.cache.pool.copy_(c.pool)
    c.check_attention(scale=6.25)


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(1, 3000)] * 3, [(5, 900), (2, 17)], [(100, 700), (30, 2000)]])
def test_calls_repeat_bit_for_bit_whatever_the_workspace_held(gpu, shapes):
    c = Call(gpu, shapes, 8, 2, 128, 64, torch.bfloat16, 59)
    first = c.check_attention()
    stream = torch.cuda.current_stream().cuda_stream
    for fill in (255, 0, 127):
        c.kernels._workspace[stream, 128][2].fill_(fill)
        assert torch.equal(c.kernels.attention(c.cache, c.sequences, c.dq, 128 ** -0.5), first)


@pytest.mark.gpu
def test_pages_shared_by_sequences_that_only_read_them(gpu):
    c = Call(gpu, [(1, 64), (1, 64), (20, 64)], 4, 2, 64, 16, torch.bfloat16, 61)
    for s in (1, 2):  # the first three pages of all are the first sequence's
        c.table[s, :3] = c.table[0, :3]
    c.sequences.page_table.copy_(c.table)
    c.check_attention()


@pytest.mark.gpu
def test_two_streams_and_a_captured_call(gpu):
    calls = [Call(gpu, shapes, 8, 2, 128, 64, torch.bfloat16, 67 + i) for i, shapes in enumerate(([(1, 5000), (1, 300)], [(40, 900), (3, 100)]))]
    kernels = calls[0].kernels
    alone = [kernels.attention(c.cache, c.sequences, c.dq, 0.1) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):  # side by side, each stream with its own workspace
        for c, stream, out in zip(calls, streams, outs):
            with torch.cuda.stream(stream):
                out.append(kernels.attention(c.cache, c.sequences, c.dq, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for out, want in zip(outs, alone) for x in out)
    # a captured append + attention, replayed with new rows, another page table and another context
    c = calls[0]
    out, q = torch.zeros_like(c.dq, memory_format=torch.contiguous_format), torch.zeros_like(c.dq, memory_format=torch.contiguous_format)

    def step():
        kernels.append(c.cache, c.sequences, c.dk, c.dv, q=c.dq, q_out=q)
        kernels.attention(c.cache, c.sequences, q, 0.1, out=out)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        step()
    pool = c.cache.pool.clone()
    for context in ([5000, 300], [4097, 0], [1, 320]):
        c.sequences.context.copy_(torch.tensor(context, dtype=torch.int32))
        if context[1] == 320:
            c.sequences.page_table.copy_(torch.randint(0, c.pool.shape[0], c.table.shape, generator=c.g))
            c.sequences.page_table[1, 4] = (c.sequences.page_table[0, 0] + 1) % c.pool.shape[0]  # appended to by one sequence only
        c.d_qkv.copy_(torch.randn(c.qkv.shape, generator=c.g))
        c.cache.pool.copy_(pool)
        graph.replay()
        got, after = out.clone(), c.cache.pool.clone()
        c.cache.pool.copy_(pool)
        step()
        assert torch.equal(out, got) and torch.equal(c.cache.pool, after) and kernels.bad_flag() == 0


@pytest.mark.gpu
def test_a_workspace_is_not_made_under_capture(gpu):
    c = Call(gpu, [(1, 20)], 4, 2, 64, 16, torch.bfloat16, 71)
    stream = torch.cuda.Stream()
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
        with pytest.raises(ValueError, match="workspace"):
            c.kernels.attention(c.cache, c.sequences, c.dq, 0.1)


@pytest.mark.gpu
def test_tensors_elsewhere_and_other_layouts_are_refused(gpu):
    c = Call(gpu, [(2, 20)], 4, 2, 64, 16, torch.bfloat16, 73)
    k, call = c.kernels, (c.cache, c.sequences)
    with pytest.raises(ValueError):  # on the CPU
        k.attention(*call, c.q, 0.1)
    with pytest.raises(ValueError):
        k.append(*call, c.k, c.v)
    with pytest.raises(ValueError):
        k.append(*call, c.dk, c.dv, q=c.dq, q_weight=torch.ones(64, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        k.qk_norm_rope(c.q, None, None)
    from padra_b200 import attention as A

    with pytest.raises(ValueError):
        k.attention(A.KvCache.over(c.pool, 16, 64), c.sequences, c.dq, 0.1)
    with pytest.raises(ValueError):
        k.read(c.cache, A.Sequences(c.table, c.begin, c.context, c.rows, 2))
    with pytest.raises(ValueError):
        k.append(*call, c.dk, c.dv, A.Rotary(torch.zeros(32, dtype=torch.float64)))
    with pytest.raises(ValueError):  # heads apart
        k.attention(*call, c.d_qkv[:, :8 * 64].unflatten(1, (8, 64))[:, ::2], 0.1)
    with pytest.raises(ValueError):
        k.attention(*call, c.dq.transpose(1, 2).contiguous().transpose(1, 2), 0.1)
    with pytest.raises(ValueError):
        k.attention(*call, c.dq[:1], 0.1)
    with pytest.raises(A.B.PadraError):  # seven heads over two
        k.attention(*call, torch.zeros((2, 7, 64), dtype=torch.bfloat16, device=gpu), 0.1)
    with pytest.raises(A.B.PadraError):
        k.attention(*call, c.dq.float(), 0.1)
    assert k.bad_flag() == 0


@pytest.mark.gpu
def test_a_flag_that_is_up_changes_nothing(gpu):
    c = Call(gpu, [(1, 700), (30, 100)], 4, 2, 64, 16, torch.bfloat16, 79)
    want = c.check_attention()
    c.kernels.bad.fill_(1)
    assert torch.equal(c.kernels.attention(c.cache, c.sequences, c.dq, 64 ** -0.5), want)
    c.kernels.append(c.cache, c.sequences, c.dk, c.dv)
    k, _ = c.kernels.read(c.cache, c.sequences, dtype=torch.float32)
    assert torch.equal(k.cpu().double(), R.dequantise(*R.quantise(c.k.double()))) and c.kernels.bad_flag() == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, heads, kv_heads, dim, interleaved", [(torch.bfloat16, 5, 3, 128, False), (torch.float32, 4, 2, 64, True), (torch.float16, 1, 1, 64, False)])
def test_rows_do_not_depend_on_how_many_share_a_call(gpu, dtype, heads, kv_heads, dim, interleaved):
    """One call for all rows against calls for 1, 40, 650 and the remaining rows: launch shapes differ, bytes do not."""
    from padra_b200 import attention as A

    total = 2900
    c = Call(gpu, [(total, total + 7)], heads, kv_heads, dim, 64, dtype, 83)
    weight = (1 + 0.3 * torch.randn(dim, generator=c.g)).bfloat16().to(gpu)
    inv_freq, amplitude = R.yarn_like(dim // 2, 2.0)
    rotary = A.Rotary(inv_freq.to(gpu), interleaved, amplitude)
    before = c.cache.pool.clone()
    q = c.kernels.append(c.cache, c.sequences, c.dk, c.dv, rotary, weight, 1e-6, c.dq, weight)
    whole = c.cache.pool.clone()
    positions = torch.arange(7, total + 7, dtype=torch.int32, device=gpu)
    q_plain, k_plain = c.kernels.qk_norm_rope(c.dq, c.dk, positions, rotary, weight, weight)
    read = c.kernels.read(c.cache, c.sequences, dtype=torch.float32)
    c.cache.pool.copy_(before)
    at = 0
    for n in (1, 40, 650, total - 691):
        part = slice(at, at + n)
        begin = torch.tensor([0, n], dtype=torch.int32, device=gpu)
        seq = A.Sequences(c.sequences.page_table, begin, torch.tensor([7 + at + n], dtype=torch.int32, device=gpu), n, n)
        assert torch.equal(c.kernels.append(c.cache, seq, c.dk[part], c.dv[part], rotary, weight, 1e-6, c.dq[part], weight), q[part])
        got = c.kernels.qk_norm_rope(c.dq[part], c.dk[part], positions[part], rotary, weight, weight)
        assert torch.equal(got[0], q_plain[part]) and torch.equal(got[1], k_plain[part])
        assert all(torch.equal(x, y[part]) for x, y in zip(c.kernels.read(c.cache, seq, dtype=torch.float32), read))
        at += n
    assert torch.equal(c.cache.pool, whole) and c.kernels.bad_flag() == 0
    # the first and the last rows against the formulas
    for r in (0, 1, 700, total - 1):
        p = torch.tensor([r + 7])
        want = R.rotate(R.rms(c.q[r:r + 1], weight.cpu(), 1e-6), p, inv_freq, interleaved, amplitude)
        slack = 2.0 ** -19 * 2 * amplitude * want.abs().amax(-1, keepdim=True) * math.sqrt(2)
        for got in (q, q_plain):  # either call rounds cos and sin its own way: near the same values, not the same bits
            assert ((got[r:r + 1].cpu().double() - want).abs() <= HALF[dtype] * want.abs() + slack).all()
        k = R.rotate(R.rms(c.k[r:r + 1], weight.cpu(), 1e-6), p, inv_freq, interleaved, amplitude)
        assert torch.equal(read[0][r:r + 1].cpu().double(), R.dequantise(*R.quantise(k)))


@pytest.mark.gpu
def test_values_on_and_beside_the_borders_of_codes(gpu):
    """Scales that are powers of two and others, values exactly between two codes and one step of FP32 to either side, scales below
    FP16's normal range: the bytes of a division in 64 bits."""
    rows = 64
    c = Call(gpu, [(rows, rows)], 1, 2, 64, 16, torch.float32, 89)
    g = torch.Generator().manual_seed(5)
    for r in range(rows):
        scale = 2.0 ** -(r % 27) * (1 if r % 2 else 1.1376953125)
        x = (torch.randint(-7, 8, (4, 64), generator=g) + torch.tensor([0.5, -0.5, 0.0, 0.5])[:, None]).clamp(-7, 7) * scale
        x[:, ::32] = 7 * scale
        x = torch.where(torch.rand(x.shape, generator=g) < 0.3, torch.nextafter(x, x * 2), torch.where(torch.rand(x.shape, generator=g) < 0.3, torch.nextafter(x, x * 0), x))
        c.k[r], c.v[r] = x[:2], x[2:]
    c.d_qkv.copy_(c.qkv)
    c.kernels.append(c.cache, c.sequences, c.dk, c.dv)
    want = c.pool.clone()
    for r in range(rows):
        for h in range(2):
            R.store(want, int(c.table[0, r // 16]), h, r % 16, 16, c.k[r, h].double(), c.v[r, h].double())
    assert torch.equal(c.cache.pool.cpu(), want) and c.kernels.bad_flag() == 0


@pytest.mark.gpu
def test_results_of_a_call_on_another_stream_are_that_streams_memory(gpu):
    """Blocks that the current stream has just given back may still be in use there: the call's results do not take them."""
    c = Call(gpu, [(1, 400), (30, 200)], 4, 2, 64, 16, torch.bfloat16, 97)
    q, side = c.dq.contiguous(), torch.cuda.Stream()
    want = c.kernels.attention(c.cache, c.sequences, q, 0.1)
    k, v = c.kernels.read(c.cache, c.sequences)
    rope = c.kernels.qk_norm_rope(q, k, None)
    torch.cuda.synchronize()
    held = [torch.empty_like(q) for _ in range(8)] + [torch.empty_like(k) for _ in range(8)]
    freed = {t.data_ptr() for t in held}
    del held
    got = (c.kernels.attention(c.cache, c.sequences, q, 0.1, stream=side), *c.kernels.read(c.cache, c.sequences, stream=side),
           *c.kernels.qk_norm_rope(q, k, None, stream=side), c.kernels.append(c.cache, c.sequences, c.dk, c.dv, q=q, stream=side))
    side.synchronize()
    assert not freed & {t.data_ptr() for t in got}
    assert all(torch.equal(x, y) for x, y in zip(got, (want, k, v, *rope, q)))


@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv_heads, dim, page", [(8, 2, 64, 16), (8, 2, 128, 64), (3, 1, 64, 32)])
@pytest.mark.parametrize("kind", ["one column block of 128", "blocks of more than 128", "both"])
def test_runs_of_many_short_units_on_one_cta(gpu, heads, kv_heads, dim, page, kind):
    """A prompt whose units are cut, then so many short ones that a CTA (one per SM) has four and more units of one to three tiles in its
    run: blocks of at most 128 columns, in which both halves work on the same columns, larger ones, and both kinds in turn."""
    g = torch.Generator().manual_seed(101 + dim)
    group, shapes = heads // kv_heads, [(200, 1500)]
    for i in range(800 // kv_heads):
        wide = kind == "blocks of more than 128" or kind == "both" and bool(torch.rand(1, generator=g) < 0.5)
        rows = int(torch.randint(128 // group + 1, 160 // group, (1,), generator=g)) if wide else int(torch.randint(1, 128 // group + 1, (1,), generator=g))
        far = i % 7 == 3  # two or three tiles now and then
        shapes.append((rows, rows + int(torch.randint(128 if far else 0, 260 if far else 128 - rows + 1, (1,), generator=g))))
    c = Call(gpu, shapes, heads, kv_heads, dim, page, torch.bfloat16, 103, spare_rows=1)
    first = c.check_attention()
    for _ in range(30):
        out = torch.full_like(first, 7.0)
        assert torch.equal(c.kernels.attention(c.cache, c.sequences, c.dq, dim ** -0.5, out=out), first)
    assert c.kernels.bad_flag() == 0


@pytest.mark.gpu
def test_two_threads_on_one_stream(gpu):
    """Calls with many cut units, whose joins read the workspace that the threads share: each gets its own results."""
    calls = [Call(gpu, shapes, 8, 2, 128, 64, torch.bfloat16, 107 + i) for i, shapes in enumerate(([(1, 3000)] * 3, [(1, 5000), (2, 900)], [(100, 700), (30, 2000)]))]
    kernels = calls[0].kernels
    alone = [kernels.attention(c.cache, c.sequences, c.dq, 0.1) for c in calls]
    torch.cuda.synchronize()
    outs, start = [[] for _ in calls], threading.Barrier(len(calls))

    def work(c, out):
        start.wait()
        for _ in range(400):
            out.append(kernels.attention(c.cache, c.sequences, c.dq, 0.1))

    threads = [threading.Thread(target=work, args=x) for x in zip(calls, outs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(kernels._workspace) == 1 and kernels.bad_flag() == 0
    for out, want in zip(outs, alone):
        assert len(out) == 400 and all(torch.equal(x, want) for x in out)


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(1, 300), (3, 40)], [(40, 300), (130, 140)]])  # few and many columns
@pytest.mark.parametrize("value, scale", [(0.0, 1e-8), (1e-38, 1e-3), (1e-38, 1e-20), (-1.0, 1e-38), (1e-30, -1e-30)])
def test_scores_too_small_for_32_bits_give_equal_weights(gpu, shapes, value, scale):
    c = Call(gpu, shapes, 8, 2, 128, 64, torch.bfloat16, 109)
    c.q[:] = value
    c.d_qkv.copy_(c.qkv)
    c.check_attention(scale=scale)
    c.check_attention(scale=scale, window=30)


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(1, 300), (3, 40)], [(40, 300), (130, 140)]])
@pytest.mark.parametrize("value, scale", [(3e38, 0.1), (1e10, 1e30), (-1e20, 1e20), (1e9, 1.0)])
def test_scores_too_large_for_32_bits_are_reported(gpu, shapes, value, scale):
    c = Call(gpu, shapes, 8, 2, 128, 64, torch.bfloat16, 113)
    c.q[:] = value
    c.d_qkv.copy_(c.qkv)
    for sign in (1, -1):
        c.kernels.attention(c.cache, c.sequences, c.dq, sign * scale)
        assert c.kernels.bad_flag() == 1
        c.kernels.reset_bad()
    a, b = 64 * 64, 64 * 8  # keys of zero: all scores are
    c.pool[:, :, a:a + b] = 0
    c.cache.pool.copy_(c.pool)
    c.check_attention(scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(1, 300), (3, 40)], [(40, 300), (130, 140)]])
@pytest.mark.parametrize("level", [-1.0, 1.0])
def test_large_scores_that_differ_by_little(gpu, shapes, level):
    """Scores of +-3.5 * 2^20 and 0 to 4 more, in the exponent of two.  Every product and sum is exact in 32 bits, so the weights are 2^(t % 5)
    up to their rounding to FP16 (2^-11, as V's) whatever the size of the scores."""
    c = Call(gpu, shapes, 8, 2, 128, 64, torch.bfloat16, 127)
    c.q[:] = 0
    c.q[:, :, 0], c.q[:, :, 32] = 2.0 ** 20 * level, 1.0
    c.d_qkv.copy_(c.qkv)
    for s, (_, ctx) in enumerate(shapes):
        for t in range(ctx):
            k = torch.zeros(128, dtype=torch.float64)
            k[0], k[32], k[33] = 3.5, t % 5, 7.0  # steps of 0.5 and 1
            page, slot = int(c.table[s, t // 64]), t % 64
            values = R.fetch(c.pool, page, 64, 128)[1]
            for h in range(2):
                R.store(c.pool, page, h, slot, 64, k, values[h, slot])
    c.cache.pool.copy_(c.pool)
    out = c.kernels.attention(c.cache, c.sequences, c.dq, math.log(2)).cpu().double()
    assert c.kernels.bad_flag() == 0
    for s, (n, ctx) in enumerate(shapes):
        v = R.tokens(c.pool, c.table[s], ctx, 64, 128)[1].repeat_interleave(4, 1)
        for r in range(n):
            seen = v[:ctx - n + r + 1]
            p = 2.0 ** (torch.arange(len(seen)) % 5).double()
            p = (p / p.sum())[:, None, None]
            want, bound = (p * seen).sum(0), 2 * 3 * 2 ** -11 * (p * seen.abs()).sum(0)
            assert ((out[int(c.begin[s]) + r] - want).abs() <= bound + 2.0 ** -8 * want.abs()).all()


def test_a_scale_that_leaves_32_bits_is_refused(lib):
    from padra_b200 import binding as B

    c, s, _ = structs(rows=0)
    p = 4096
    for scale, want in ((3e38, B.INVALID_ARGUMENT), (-3e38, B.INVALID_ARGUMENT), (2e38, B.OK)):
        assert lib.padra_attention_q4(C.byref(c), C.byref(s), p, p, 512, 512, 4, 0, scale, 0, p, 1 << 40, p, None) == want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim, interleaved", [(64, False), (128, True), (256, False)])
@pytest.mark.parametrize("eps", [1e-6, 1e-30, 0.0])
def test_norm_of_values_whose_squares_leave_32_bits(gpu, dtype, dim, interleaved, eps):
    """Heads of ordinary size among others up to 1e38 and down to 1e-38: each as its formula gives it, whatever its neighbours are."""
    from padra_b200 import attention as A

    g = torch.Generator().manual_seed(131 + dim)
    rows, heads = 9, 7
    x = torch.randn((rows, heads, dim), generator=g).double()
    size = torch.tensor([1.0, 1e18, 1e20, 1e36, 1e-19, 1e-25, 1e-36], dtype=torch.float64)
    plain = x.to(dtype)
    x = (x * size[torch.stack([torch.randperm(7, generator=g) for _ in range(rows)])][..., None]).to(dtype)
    weight = (1 + 0.3 * torch.randn(dim, generator=g)).bfloat16()
    inv_freq, amplitude = R.yarn_like(dim // 2, 2.0)
    positions = torch.arange(rows, dtype=torch.int32)
    kernels, rotary = A.AttentionKernels(gpu), A.Rotary(inv_freq.to(gpu), interleaved, amplitude)
    got = kernels.qk_norm_rope(x.to(gpu), x.to(gpu), positions.to(gpu), rotary, weight.to(gpu), weight.to(gpu), eps)
    normed = R.rms(x, weight, eps)
    want = R.rotate(normed, positions, inv_freq, interleaved, amplitude)
    # as in test_norm_and_rotation; a BF16 value below the normal range is off by half a step of 2^-133
    slack = 2.0 ** -19 * 2 * amplitude * normed.abs().amax(-1, keepdim=True) + 2.0 ** -134
    for y in got:
        assert ((y.cpu().double() - want).abs() <= HALF[dtype] * want.abs() + slack).all()
    assert kernels.bad_flag() == 0
    # an ordinary head's bits do not depend on what lies beside it
    alone = kernels.qk_norm_rope(plain.to(gpu), None, positions.to(gpu), rotary, weight.to(gpu), None, eps)[0]
    same = (x == plain).all(-1)
    assert same.any() and torch.equal(got[0].cpu()[same], alone.cpu()[same])
    if dim < 256:  # the queries of an append
        begin, context = torch.tensor([0, rows], dtype=torch.int32, device=gpu), torch.tensor([rows], dtype=torch.int32, device=gpu)
        cache = A.KvCache(1, 16, 1, dim, gpu)
        k = torch.ones((rows, 1, dim), dtype=dtype, device=gpu)
        q = kernels.append(cache, A.Sequences(torch.zeros((1, 1), dtype=torch.int32, device=gpu), begin, context, rows, rows), k, k, rotary, weight.to(gpu), eps, x.to(gpu), weight.to(gpu))
        assert ((q.cpu().double() - want).abs() <= HALF[dtype] * want.abs() + slack * math.sqrt(2)).all() and kernels.bad_flag() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(5, 2), (1, 40), (7, 3)], [(60, 10), (40, 300), (5, 0)]])  # more rows than context: few and many columns
@pytest.mark.parametrize("window", [2 ** 40 + 1, 2 ** 31 - 1, 2 ** 31 - 8, 2 ** 30])
def test_a_window_wider_than_any_context_is_none(gpu, shapes, window):
    c = Call(gpu, shapes, 8, 2, 64, 16, torch.bfloat16, 137)
    assert torch.equal(c.check_attention(window=window), c.check_attention())


@pytest.mark.gpu
def test_calls_without_rows(gpu):
    c = Call(gpu, [(0, 30), (0, 0)], 8, 2, 64, 16, torch.bfloat16, 139, strided=False)
    k, before = c.kernels, c.cache.pool.clone()
    from padra_b200 import attention as A

    rotary = A.Rotary(torch.ones(32, dtype=torch.float64, device=gpu))
    empty = lambda heads: torch.empty((0, heads, 64), dtype=torch.bfloat16, device=gpu)  # noqa: E731
    assert k.attention(c.cache, c.sequences, empty(8), 0.1).shape == (0, 8, 64)
    assert k.append(c.cache, c.sequences, empty(2), empty(2), rotary, q=empty(8)).shape == (0, 8, 64)
    assert k.append(c.cache, c.sequences, empty(2), empty(2)) is None
    assert [x.shape for x in k.read(c.cache, c.sequences)] == [(0, 2, 64)] * 2
    assert [x.shape for x in k.qk_norm_rope(empty(8), empty(2), torch.empty(0, dtype=torch.int32, device=gpu), rotary)] == [(0, 8, 64), (0, 2, 64)]
    none = A.Sequences(torch.empty((0, 3), dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu), torch.empty(0, dtype=torch.int32, device=gpu), 0, 0)
    assert k.attention(c.cache, none, empty(8), 0.1).shape == (0, 8, 64)
    assert torch.equal(c.cache.pool, before) and k.bad_flag() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim, page", [(64, 64), (128, 16)])
@pytest.mark.parametrize("heads, kv_heads, rows, context", MARKED)
def test_no_tile_of_a_split_sequence_is_lost_or_doubled(gpu, dtype, dim, page, heads, kv_heads, rows, context):
    c = Call(gpu, [(rows, context)], heads, kv_heads, dim, page, dtype, 149)
    k, v, want = R.marked(rows, context, dim)
    R.fill(c.pool, c.table[0], page, *(x[:, None].expand(-1, kv_heads, -1) for x in (k, v)))
    c.cache.pool.copy_(c.pool)
    for scale, q in ((math.log(2), 1.0), (0.0, 3.0)):
        c.dq[:] = 0
        c.dq[:, :, 0] = q
        out = c.kernels.attention(c.cache, c.sequences, c.dq, scale).cpu().double()
        if not scale:  # all weights equal
            seen = (torch.arange(context) <= torch.arange(context - rows, context)[:, None]).double()
            want = seen @ v / seen.sum(1, keepdim=True)
        assert ((out - want[:, None]).abs() <= marked_bound(want, dtype)[:, None]).all()
    assert c.kernels.bad_flag() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [1, 12])
@pytest.mark.parametrize("dim", [64, 128])
def test_weights_of_fp16_rows_keep_their_low_bits(gpu, heads, dim):
    """16 tokens of weight 2^-0.30005 and value 4 against 13 of weight 1 and value -4 leave 1/2600 of the terms: FP16 weights alone, the
    first of which would be off by 0.00026, would be half of that away.  What is left: the exponential (2^-22), its argument (2^-22) and the
    rest's own rounding (2^-22) of terms that add up to 2, then the output's."""
    c = Call(gpu, [(1, 29)], heads, 1, dim, 16, torch.float16, 151)
    k, v = torch.zeros((29, 1, dim), dtype=torch.float64), torch.zeros((29, 1, dim), dtype=torch.float64)
    light = torch.arange(29) % 9 < 5
    assert int(light.sum()) == 17
    light[28] = False
    k[light, 0, 0], k[:, 0, 1] = -1.0, 7.0
    v[:] = torch.where(light, 4.0, -4.0)[:, None, None]
    v[:, :, ::32] = 7.0  # the groups' scale is one
    R.fill(c.pool, c.table[0], 16, k, v)
    c.cache.pool.copy_(c.pool)
    c.dq[:] = 0
    c.dq[:, :, 0] = 0.3
    weight = torch.where(light, 2.0 ** -float(torch.tensor(0.3).half()), 1.0).double()
    want = weight @ v[:, 0] / weight.sum()
    got = c.kernels.attention(c.cache, c.sequences, c.dq, math.log(2)).cpu().double()
    assert want[1].abs() < 1e-3 and ((got - want).abs() <= HALF[torch.float16] * want.abs() + 7 * 4 * 2.0 ** -22).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv_heads", [(8, 2), (8, 8)])
@pytest.mark.parametrize("shapes", [
    [(1, 9000), (512, 3000), (1, 40), (1, 17000), (1, 1)], [(1, 700)] * 40 + [(130, 130), (5, 6000)], [(40, 8000), (200, 200), (0, 50), (1, 8001), (33, 1000)]])
def test_prompt_chunks_beside_decode_rows(gpu, heads, kv_heads, shapes):
    """One call for rows of all kinds; every sequence tells which tokens its rows have seen."""
    c = Call(gpu, shapes, heads, kv_heads, 64, 32, torch.bfloat16, 157, spare_rows=2)
    wanted = []
    for s, (n, ctx) in enumerate(shapes):
        k, v, want = R.marked(n, ctx, 64)
        R.fill(c.pool, c.table[s], 32, *(x[:, None].expand(-1, kv_heads, -1) for x in (k, v)))
        wanted.append(want)
    c.cache.pool.copy_(c.pool)
    c.dq[:] = 0
    c.dq[:, :, 0] = 1
    out = torch.full((c.rows, heads, 64), 7.0, dtype=torch.bfloat16, device=gpu)
    c.kernels.attention(c.cache, c.sequences, c.dq, math.log(2), out=out)
    got, want = out.cpu().double(), torch.cat(wanted)
    assert ((got[:-2] - want[:, None]).abs() <= marked_bound(want, torch.bfloat16)[:, None]).all()
    assert (got[-2:] == 7).all() and c.kernels.bad_flag() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [1, 60, 140])
@pytest.mark.parametrize("first", [2, 130, 258])
def test_weights_outlast_a_large_rise_of_the_maximum(gpu, dtype, dim, rows, first):
    """Scores (in the exponent of two) of 0, then 7 for one token, the only one with a value, then 25 for another of its tile: the value's
    weight is 2^-18 of the largest, far above what FP16 weights lose, and everything is exact but the output's rounding.  160 equal
    units, so that some of them lie whole in one CTA's run."""
    c = Call(gpu, [(rows, 600)] * 20, 8, 8, dim, 64, dtype, 163)
    k, v = torch.zeros((600, dim), dtype=torch.float64), torch.zeros((600, dim), dtype=torch.float64)
    k[:, 4] = 7.0  # the groups' scale is one
    k[first, 0], v[first] = 7.0, 7.0
    k[first + 68, :4] = torch.tensor([7.0, 7.0, 7.0, 4.0])
    for s in range(20):
        R.fill(c.pool, c.table[s], 64, *(x[:, None].expand(-1, 8, -1) for x in (k, v)))
    c.cache.pool.copy_(c.pool)
    c.dq[:] = 0
    c.dq[:, :, :4] = 1
    out = c.kernels.attention(c.cache, c.sequences, c.dq, math.log(2)).cpu().double()
    weight = 2.0 ** k[:, :4].sum(1)
    for r in range(rows):
        want = 7 * weight[first] / weight[:600 - rows + r + 1].sum()
        assert ((out[r::rows] - want).abs() <= marked_bound(want, dtype) + (2.0 ** -25 if dtype == torch.float16 else 0)).all()
    assert c.kernels.bad_flag() == 0
