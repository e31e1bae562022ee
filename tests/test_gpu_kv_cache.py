"""The paged key/value cache on the GPU: rows written, read back and attended to, against plain 64-bit restatements
(tests/kv_reference.py) and, for Q8_0, against the oracle's row quantizer bit for bit."""

import ctypes

import numpy as np
import pytest

import kv_reference as ref
from conftest import load_package

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b200():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return load_package()


@pytest.fixture(scope="module")
def ctx(b200):
    c = b200.Context(0)
    yield c
    c.close()


def cu(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def fields(b200, cache, data):
    """The cache's arrays as torch views of `data` (the documented layout)."""
    import math

    import torch

    c = cache.s
    rows = [c.n_pages, c.n_kv_head, c.page_size]
    kind = torch.int8 if c.type == b200.Q8_0 else torch.float16
    shapes = [(rows + [c.head_dim], kind)] * 2 + ([(rows + [c.head_dim // 32], torch.float16)] * 2 if c.type == b200.Q8_0 else [])
    out = []
    for (shape, kind), off in zip(shapes, c.field_off):
        n = math.prod(shape) * (1 if kind == torch.int8 else 2)
        out.append(data[off:off + n].view(kind).view(shape))
    return out


class Pool:
    """A cache with `lens` sequences of random pages, everything around them filled with what must not be seen."""

    def __init__(self, b200, ctx, qtype, Hkv, D, page, lens, seed=0, spare=3, width=None):
        import torch

        rng = np.random.default_rng(seed)
        self.b200, self.ctx, self.qtype, self.Hkv, self.D, self.page, self.lens = b200, ctx, qtype, Hkv, D, page, list(lens)
        need = [-(-n // page) for n in lens]
        self.width = max([1] + need) + 1 if width is None else width
        n_pages = sum(need) + spare
        self.data = torch.zeros(ctx.L.b200_kv_cache_nbytes(qtype, Hkv, D, page, n_pages), dtype=torch.uint8, device="cuda")
        self.cache = ctx.kv_cache(qtype, Hkv, D, page, n_pages, data=self.data)
        self.f = fields(b200, self.cache, self.data)
        for a in self.f:  # unused places: NaN where the type has one, and its largest values
            a.fill_(-128 if a.dtype == torch.int8 else float("nan"))
        order = rng.permutation(n_pages)
        self.table_np = np.full((len(lens), self.width), -7, np.int32)  # entries past a sequence are not read
        at = 0
        for s, n in enumerate(need):
            self.table_np[s, :n] = order[at:at + n]
            at += n
        self.table, self.lens_t = cu(self.table_np), cu(np.array(lens, np.int32))
        self.rng = rng

    def fill(self, spread=1.0):
        """Writes every sequence's rows (through kv_write, all at once: shorter ones start at a negative position)."""
        n = max(1, max(self.lens))
        self.k = self.rng.normal(0, 1, (len(self.lens), n, self.Hkv, self.D)).astype(np.float32)
        self.v = self.rng.normal(0, spread, (len(self.lens), n, self.Hkv, self.D)).astype(np.float32)
        self.ctx.kv_write(self.cache, cu(self.k), cu(self.v), self.table, self.lens_t)
        return self

    def rows(self, s):
        """Sequence s's keys and values [len][Hkv][D] as the cache holds them, taken from its memory."""
        out = []
        for which in (0, 1):
            x = self.f[which].cpu().numpy().astype(np.float64)
            if self.qtype == self.b200.Q8_0:
                x = x * np.repeat(self.f[2 + which].cpu().numpy().astype(np.float64), 32, -1)
            n = self.lens[s]
            pos = np.arange(n)
            out.append(x[self.table_np[s, pos // self.page], :, pos % self.page] if n else np.zeros((0, self.Hkv, self.D)))
        return out

    def check_attention(self, H, n_tok, scale=None, q=None, out=None):
        scale = 1.0 / np.sqrt(self.D) if scale is None else scale
        q = self.rng.normal(0, 1.5, (len(self.lens), n_tok, H, self.D)).astype(np.float32) if q is None else q
        got = self.ctx.kv_attention(self.cache, cu(q), self.table, self.lens_t, scale, out=out)
        self.ctx.synchronize()
        kv = [self.rows(s) for s in range(len(self.lens))]
        want, tol = ref.attention(q, [k for k, _ in kv], [v for _, v in kv], self.lens, scale)
        got = got.cpu().numpy()
        assert np.isfinite(got).all()
        off = np.abs(got - want) - tol
        assert off.max() <= 0, f"{(off > 0).sum()} of {off.size} outside the bound, worst {np.max((np.abs(got - want)) / (tol + 1e-30)):.2f} of it"
        return got


# ---- refusals ----------------------------------------------------------------------------------------------------------


def test_refusals(b200, ctx):
    import torch

    with pytest.raises(b200.B200Error, match="UNSUPPORTED"):
        ctx.kv_cache(b200.Q4_K, 8, 128, 16, 4)
    with pytest.raises(b200.B200Error, match="UNSUPPORTED"):
        ctx.kv_cache(b200.F16, 8, 128, 24, 4)
    with pytest.raises(b200.B200Error, match="too few bytes"):
        ctx.kv_cache(b200.F16, 8, 128, 16, 4, data=torch.zeros(1000, dtype=torch.uint8, device="cuda"))
    with pytest.raises(b200.B200Error, match="16-byte"):
        ctx.kv_cache(b200.F16, 1, 64, 16, 1, data=torch.zeros(8192, dtype=torch.uint8, device="cuda")[1:])
    cache = ctx.kv_cache(b200.F16, 2, 64, 16, 4)
    table, lens = cu(np.zeros((2, 2), np.int32)), cu(np.array([1, 1], np.int32))
    x = torch.zeros(2, 1, 2, 64, device="cuda")
    with pytest.raises(ValueError):
        ctx.kv_write(cache, x, x[:1], table, lens)
    with pytest.raises(ValueError):
        ctx.kv_write(cache, x.half(), x.half(), table, lens)
    with pytest.raises(ValueError):
        ctx.kv_write(cache, x, x, table, lens.long())
    with pytest.raises(ValueError):
        ctx.kv_write(cache, x, x, table[:1], lens)
    with pytest.raises(ValueError):  # heads apart from each other
        ctx.kv_write(cache, x, torch.zeros(2, 1, 4, 64, device="cuda")[:, :, ::2], table, lens)
    with pytest.raises(ValueError):  # rows at two strides
        ctx.kv_write(cache, *(torch.zeros(2, 3, 2, 64, device="cuda")[:, :2] for _ in range(2)), table, lens)
    with pytest.raises(ValueError):  # one row read as many
        ctx.kv_attention(cache, x[:, :, :1].expand(2, 1, 4, 64), table, lens, 1.0)
    with pytest.raises(b200.B200Error, match="multiple of n_kv_head"):
        ctx.kv_attention(cache, torch.zeros(2, 1, 3, 64, device="cuda"), table, lens, 1.0)
    with pytest.raises(b200.B200Error, match="more than 16"):
        ctx.kv_attention(cache, torch.zeros(2, 17, 2, 64, device="cuda"), table, lens, 1.0)
    with pytest.raises(ValueError):
        ctx.kv_attention(cache, x, table, lens, 1.0, out=torch.zeros(2, 1, 2, 32, device="cuda"))
    other = b200.Context(0)
    with pytest.raises(ValueError, match="another context"):
        other.kv_write(cache, x, x, table, lens)
    other.close()
    L, vp = ctx.L, x.data_ptr()
    args = (ctx.h, None, cache.ref, table.data_ptr(), 2, lens.data_ptr())
    assert L.b200_kv_write(*args, -1, 1, vp, 128, vp, 128) == b200.ERR_INVALID
    assert L.b200_kv_write(*args, 2, 1, vp, 127, vp, 128) == b200.ERR_INVALID
    assert L.b200_kv_write(*args, 2, 1, vp + 2, 128, vp, 128) == b200.ERR_INVALID
    assert L.b200_kv_write(*args, 1 << 20, 1 << 20, vp, 128, vp, 128) == b200.ERR_INVALID
    assert L.b200_kv_write(ctx.h, None, cache.ref, table.data_ptr(), 1 << 30, lens.data_ptr(), 2, 1, vp, 128, vp, 128) == b200.ERR_INVALID
    assert L.b200_kv_write(ctx.h, None, cache.ref, None, 2, lens.data_ptr(), 2, 1, vp, 128, vp, 128) == b200.ERR_INVALID
    assert L.b200_kv_write(ctx.h, None, cache.ref, table.data_ptr() + 2, 2, lens.data_ptr(), 2, 1, vp, 128, vp, 128) == b200.ERR_INVALID
    assert L.b200_kv_read(ctx.h, None, cache.ref, table.data_ptr(), 2, lens.data_ptr(), lens.data_ptr() + 1, 2, 1, b200.F32, vp, vp) == b200.ERR_INVALID
    for name, value in (("page_size", 0), ("head_dim", 100), ("n_pages", 1 << 40), ("type", b200.F32), ("n_kv_head", 0), ("device", 1)):
        bad = b200.KvCacheStruct.from_buffer_copy(cache.s)
        setattr(bad, name, value)
        call = (ctx.h, None, ctypes.byref(bad), table.data_ptr(), 2, lens.data_ptr(), 2, 1)
        assert L.b200_kv_write(*call, vp, 128, vp, 128) == b200.ERR_INVALID
        assert L.b200_kv_attention(*call, 2, vp, 128, 1.0, vp, None, 0) == b200.ERR_INVALID
    assert L.b200_kv_read(*args, None, 2, 1, b200.Q8_0, vp, vp) == b200.ERR_UNSUPPORTED
    assert L.b200_kv_read(*args, None, 2, 1, b200.F32, vp, None) == b200.ERR_INVALID
    assert L.b200_kv_attention(*args, 2, 1, 2, vp, 64, 1.0, vp, None, 0) == b200.ERR_INVALID
    ctx.kv_write(cache, x[:0], x[:0], table[:0], lens[:0])
    assert ctx.kv_attention(cache, x[:0], table[:0], lens[:0], 1.0).shape == (0, 1, 2, 64)
    cache.close()
    with pytest.raises(ValueError, match="closed"):
        ctx.kv_write(cache, x, x, table, lens)
    ctx.synchronize()


@pytest.mark.parametrize("qname", ["F16", "Q8_0"])
def test_caches_that_are_not_laid_out_as_documented_are_refused(b200, ctx, qname):
    """Arrays that the struct places elsewhere, or memory that is not aligned, would be read past their ends or misaligned."""
    import torch

    cache = ctx.kv_cache(getattr(b200, qname), 2, 64, 16, 4)
    table, lens, x = cu(np.zeros((1, 2), np.int32)), cu(np.array([1], np.int32)), torch.zeros(1, 1, 2, 64, device="cuda").data_ptr()
    kinds = [("data", cache.s.data + 8), ("data", cache.s.data + 1), ("data", 0), ("nbytes", cache.s.nbytes - 1)]
    kinds += [(i, cache.s.field_off[i] + by) for i in range(4) for by in (-256, -16, 1, 16, 1 << 40)]
    for name, value in kinds:
        bad = b200.KvCacheStruct.from_buffer_copy(cache.s)
        if name in ("data", "nbytes"):
            setattr(bad, name, value)
        else:
            bad.field_off[name] = value
        call = (ctx.h, None, ctypes.byref(bad), table.data_ptr(), 2, lens.data_ptr())
        assert ctx.L.b200_kv_write(*call, 1, 1, x, 128, x, 128) == b200.ERR_INVALID
        assert ctx.L.b200_kv_read(*call, None, 1, 1, b200.F32, x, x) == b200.ERR_INVALID
        assert ctx.L.b200_kv_attention(*call, 1, 1, 2, x, 128, 1.0, x, None, 0) == b200.ERR_INVALID
    cache.close()
    ctx.synchronize()


def test_bad_pages_and_lengths_are_reported_and_left_out(b200, ctx):
    import torch

    p = Pool(b200, ctx, b200.F16, 2, 64, 16, [40, 20, 33], seed=3).fill()
    ctx.synchronize()
    before = p.data.clone()
    x = torch.ones(3, 1, 2, 64, device="cuda")
    for bad_len in (-1, p.width * 16 + 1, 2**31 - 1, -(2**31)):
        lens = p.lens_t.clone()
        lens[1] = bad_len
        q = torch.ones(3, 1, 2, 64, device="cuda")
        out = ctx.kv_attention(p.cache, q, p.table, lens, 1.0)
        with pytest.raises(b200.B200Error, match="RANGE"):
            ctx.synchronize()
        assert not out[1].any() and out[0].any() and out[2].any()
        lens[0] = lens[2] = 0
        ctx.kv_write(p.cache, x, x, p.table, lens)
        k, v = ctx.kv_read(p.cache, p.table, lens, n_tok=5)
        with pytest.raises(b200.B200Error, match="RANGE"):
            ctx.synchronize()
        assert torch.equal(p.data, before) and not k.any() and not v.any()
    for bad in (-1, p.cache.s.n_pages, 2**31 - 1, -(2**31)):
        table = p.table.clone()
        table[0, 1] = bad  # positions 16 to 31 of sequence 0
        q = p.rng.normal(0, 1, (3, 1, 4, 64)).astype(np.float32)
        out = ctx.kv_attention(p.cache, cu(q), table, p.lens_t, 0.125).cpu().numpy()
        k, v = ctx.kv_read(p.cache, table, p.lens_t, n_tok=40)
        with pytest.raises(b200.B200Error, match="RANGE"):
            ctx.synchronize()
        kk, vv = p.rows(0)
        keep = np.r_[0:16, 32:40]
        for h in range(4):
            want, tol = ref.softmax_attention(q[0, 0, h], kk[keep, h // 2], vv[keep, h // 2], 0.125)
            assert (np.abs(out[0, 0, h] - want) <= tol).all()
        assert np.array_equal(k[0].cpu().numpy()[keep], kk[keep]) and not k[0, 16:32].any() and not v[0, 16:32].any()
        ctx.kv_write(p.cache, torch.ones(3, 24, 2, 64, device="cuda")[:1], torch.ones(1, 24, 2, 64, device="cuda"), table[:1], p.lens_t[:1])
        with pytest.raises(b200.B200Error, match="RANGE"):
            ctx.synchronize()
        assert torch.equal(p.f[0][p.table_np[0, 1]], fields(b200, p.cache, before)[0][p.table_np[0, 1]])
        p.data.copy_(before)


def test_an_error_on_another_stream_is_reported_once(b200, ctx, oracle):
    """A bad length on a side stream, recorded before, while or after the context reports an error of its own: whichever
    report comes after it names it."""
    import torch

    p = Pool(b200, ctx, b200.F16, 1, 64, 16, [20], seed=26).fill()
    q, out, bad = torch.ones(1, 1, 1, 64, device="cuda"), torch.empty(1, 1, 1, 64, device="cuda"), cu(np.array([-1], np.int32))
    w = ctx.weight(b200.Q8_0, 64, 4, data=oracle.quantize(b200.Q8_0, np.ones((4, 64), np.float32)))
    ids = cu(np.array([9], np.int32))
    side = torch.cuda.Stream()
    ctx.synchronize()
    torch.cuda.synchronize()

    def report():
        return "" if ctx.L.b200_synchronize(ctx.h) == b200.OK else ctx.L.b200_last_error(ctx.h).decode()

    for i in range(400):
        ctx.get_rows(w, ids)
        with torch.cuda.stream(side):
            torch.cuda._sleep(500 * i)  # up to some 100 us
            ctx.kv_attention(p.cache, q, p.table, bad, 1.0, out=out)
        first = report()
        side.synchronize()
        second = report()
        assert "get_rows" in first and "get_rows" not in second, i
        assert ("kv cache" in first) + ("kv cache" in second) == 1, i
    ctx.free_weight(w)


# ---- write and read ----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("Hkv,page,lens", [(1, 16, [1]), (8, 16, [5, 0, 33]), (3, 48, [48, 49, 1, 130]), (5, 64, [7])])
def test_q8_0_rows_are_the_oracles_bit_for_bit(b200, ctx, oracle, D, Hkv, page, lens):
    p = Pool(b200, ctx, b200.Q8_0, Hkv, D, page, lens, seed=D + Hkv)
    n = max(lens)
    k = (p.rng.normal(0, 1, (len(lens), n, Hkv, D)) * 10.0 ** p.rng.integers(-6, 4, (len(lens), n, Hkv, 1))).astype(np.float32)
    v = p.rng.normal(0, 1, (len(lens), n, Hkv, D)).astype(np.float32)
    k[0, -1, 0, :32] = 0.0
    v[0, -1, 0, 32:64] = np.arange(-16, 16) / 2  # ties
    before = p.data.clone()
    ctx.kv_write(p.cache, cu(k), cu(v), p.table, p.lens_t)
    ctx.synchronize()
    want = [f.cpu().numpy().copy() for f in fields(b200, p.cache, before)]
    for which, x in ((0, k), (1, v)):
        blocks = oracle.quantize(b200.Q8_0, x.reshape(-1, D)).reshape(len(lens), n, Hkv, D // 32, 34)
        for s, size in enumerate(lens):
            for pos in range(size):
                r = n - size + pos
                at = p.table_np[s, pos // page], slice(None), pos % page
                want[which][at] = blocks[s, r, :, :, 2:].reshape(Hkv, D).view(np.int8)
                want[2 + which][at] = np.ascontiguousarray(blocks[s, r, :, :, :2]).view(np.float16)[..., 0]
    for got, w in zip(p.f, want):
        assert np.array_equal(got.cpu().numpy().view(np.uint8), w.view(np.uint8))  # other places included


@pytest.mark.parametrize("D,Hkv,page,lens", [(64, 1, 16, [1]), (128, 8, 16, [5, 0, 33]), (96, 3, 48, [48, 49, 1, 130]), (256, 2, 4096, [100, 3])])
def test_f16_rows_are_rounded_once(b200, ctx, D, Hkv, page, lens):
    p = Pool(b200, ctx, b200.F16, Hkv, D, page, lens, seed=D)
    before = [f.cpu().numpy().copy() for f in p.f]
    p.fill()
    ctx.synchronize()
    n = max(lens)
    for which, x in ((0, p.k), (1, p.v)):
        for s, size in enumerate(lens):
            for pos in range(size):
                before[which][p.table_np[s, pos // page], :, pos % page] = x[s, n - size + pos].astype(np.float16)
        assert np.array_equal(p.f[which].cpu().numpy().view(np.uint16), before[which].view(np.uint16))


def test_rows_of_a_fused_product_are_taken_as_they_lie(b200, ctx):
    """k and v are columns of one q|k|v product: strided rows, aligned and not (the columns' offset is odd)."""
    import torch

    for qtype in (b200.F16, b200.Q8_0):
        for extra in (256, 1):
            a, b = (Pool(b200, ctx, qtype, 2, 64, 16, [9, 20], seed=1).fill() for _ in range(2))
            wide = cu(a.rng.normal(0, 1, (2 * 7, extra + 2 * 128)).astype(np.float32))
            k, v = wide[:, extra:extra + 128].view(2, 7, 2, 64), wide[:, extra + 128:].view(2, 7, 2, 64)
            a.ctx.kv_write(a.cache, k, v, a.table, a.lens_t)
            b.ctx.kv_write(b.cache, k.contiguous(), v.contiguous(), b.table, b.lens_t)
            ctx.synchronize()
            assert torch.equal(a.data, b.data)
            q = wide[:, extra:extra + 256].view(2, 7, 4, 64)
            assert torch.equal(ctx.kv_attention(a.cache, q, a.table, a.lens_t, 0.1), ctx.kv_attention(a.cache, q.contiguous(), a.table, a.lens_t, 0.1))


@pytest.mark.parametrize("qname", ["F16", "Q8_0"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("D,Hkv,page,lens,start,n", [
    (64, 1, 16, [1], None, 1), (128, 8, 16, [5, 0, 33], None, 40), (128, 8, 16, [5, 0, 33], [4, 3, 15], 17), (96, 3, 48, [48, 49, 1, 130], [47, 48, 9, 0], 2),
    (256, 2, 32, [100, 3], [-5, 1], 9),
])
def test_rows_read_back(b200, ctx, qname, half, D, Hkv, page, lens, start, n):
    import torch

    p = Pool(b200, ctx, getattr(b200, qname), Hkv, D, page, lens, seed=n).fill()
    kind = torch.float16 if half else torch.float32
    shape = (len(lens), n, Hkv, D)
    for shift in (0, 1):  # aligned outputs, and outputs at an odd element
        buf = torch.full((2, int(np.prod(shape)) + 1), 7.0, dtype=kind, device="cuda")
        k, v = (buf[i, shift:shift + int(np.prod(shape))].view(shape) for i in (0, 1))
        ctx.kv_read(p.cache, p.table, p.lens_t, start=None if start is None else cu(np.array(start, np.int32)), k=k, v=v)
        ctx.synchronize()
        for s, size in enumerate(lens):
            want = p.rows(s)
            for r in range(n):
                pos = (start[s] if start else 0) + r
                for got, w in zip((k, v), want):
                    row = got[s, r].cpu().numpy()
                    if 0 <= pos < size:
                        assert np.array_equal(row, w[pos].astype(np.float32).astype(row.dtype))
                    else:
                        assert (row == 7.0).all()  # left as it was


# ---- attention ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("qname", ["F16", "Q8_0"])
@pytest.mark.parametrize("D,Hkv,group,page,n_tok,lens", [
    (128, 8, 2, 16, 1, [517]),
    (128, 2, 1, 16, 1, [1, 2, 15, 16, 17, 31, 32, 33]),
    (128, 8, 2, 32, 5, [1, 5, 300, 64, 0, 4, 65, 127]),      # rows of a verify step, some before the sequence's start
    (64, 3, 5, 48, 2, [777, 1, 0, 48, 49, 600, 95]),
    (64, 1, 7, 64, 16, [200, 16, 15]),
    (96, 2, 3, 16, 1, [100, 1000]),
    (96, 1, 16, 80, 3, [81, 333]),
    (256, 2, 4, 32, 1, [260, 31]),
    (256, 1, 8, 16, 4, [100, 3]),
    (128, 1, 64, 128, 1, [129, 128]),
    (128, 4, 8, 16, 2, [2500]),
    (128, 2, 2, 4096, 1, [4097, 100]),
])
def test_attention(b200, ctx, qname, D, Hkv, group, page, n_tok, lens):
    import torch

    p = Pool(b200, ctx, getattr(b200, qname), Hkv, D, page, lens, seed=len(lens) + D).fill()
    out = torch.full((len(lens), n_tok, Hkv * group, D), float("nan"), device="cuda")
    got = p.check_attention(Hkv * group, n_tok, out=out)
    for s, n in enumerate(lens):  # rows that see nothing
        assert not got[s, :max(0, n_tok - n)].any()


@pytest.mark.parametrize("qname", ["F16", "Q8_0"])
def test_attention_is_split_over_a_long_cache(b200, ctx, qname):
    """One sequence, one key/value head: the length is all there is to spread over the GPU; and many lengths at once."""
    Pool(b200, ctx, getattr(b200, qname), 1, 128, 64, [60000], seed=5).fill().check_attention(2, 1)
    Pool(b200, ctx, getattr(b200, qname), 2, 64, 16, [9000, 1, 3000, 0, 17, 5000, 40, 2600], seed=6).fill().check_attention(4, 2)


@pytest.mark.parametrize("qname", ["F16", "Q8_0"])
@pytest.mark.parametrize("D,Hkv,group,page,n_tok,lens", [
    (64, 3, 5, 48, 2, [777, 1, 0, 48, 49, 600, 95]),
    (64, 2, 2, 16, 1, [130, 5]),
    (96, 2, 3, 16, 1, [100, 1000, 0]),
    (96, 1, 4, 80, 4, [81, 333, 2]),
    (128, 8, 2, 32, 5, [1, 5, 300, 64, 0, 4, 65, 127]),
    (128, 2, 1, 16, 1, [1, 2, 15, 16, 17, 31, 32, 33]),
    (128, 1, 20, 16, 2, [400, 64]),
    (256, 2, 4, 32, 3, [260, 31, 1]),
])
def test_attention_with_a_wide_table(b200, ctx, qname, D, Hkv, group, page, n_tok, lens):
    """The same with a table that allows long sequences: the work is cut by positions and joined by a second kernel."""
    import torch

    p = Pool(b200, ctx, getattr(b200, qname), Hkv, D, page, lens, seed=D + len(lens), width=-(-5000 // page)).fill()
    assert ctx.L.b200_kv_attention_workspace(ctx.h, p.cache.ref, p.width, len(lens), n_tok, Hkv * group) > 0
    out = torch.full((len(lens), n_tok, Hkv * group, D), float("nan"), device="cuda")
    got = p.check_attention(Hkv * group, n_tok, out=out)
    for s, n in enumerate(lens):
        assert not got[s, :max(0, n_tok - n)].any()


def test_attention_of_many_sequences(b200, ctx):
    """More sequences than a CTA has threads: their lengths are scanned in several steps."""
    rng = np.random.default_rng(20)
    lens = rng.integers(0, 40, 300).tolist()
    lens[131] = 5000
    Pool(b200, ctx, b200.F16, 1, 64, 16, lens, seed=20).fill().check_attention(2, 1)


@pytest.mark.parametrize("qname,D,Hkv,group,n_tok", [("F16", 64, 3, 2, 1), ("Q8_0", 128, 3, 4, 3), ("F16", 256, 2, 1, 2)])
@pytest.mark.parametrize("where", [0, 131, 299])
def test_attention_of_more_items_than_ctas(b200, ctx, qname, D, Hkv, group, n_tok, where):
    """Many short sequences, empty ones among them, and a long one that many CTAs share: a CTA ends items that others began,
    takes some whole, and begins at most one that others end."""
    import torch

    lens = np.random.default_rng(23).integers(0, 100, 300).tolist()
    lens[7] = lens[298] = 0
    lens[where] = 4500
    p = Pool(b200, ctx, getattr(b200, qname), Hkv, D, 16, lens, seed=23)
    short = p.rng.normal(0, 1, (2, 300, 100, Hkv, D)).astype(np.float32)
    row = p.rng.normal(0, 1, (2, 1, 4500, Hkv, D)).astype(np.float32)
    ctx.kv_write(p.cache, cu(short[0]), cu(short[1]), p.table, p.lens_t)
    ctx.kv_write(p.cache, cu(row[0]), cu(row[1]), cu(p.table_np[where:where + 1]), cu(np.array([4500], np.int32)))
    q = p.rng.normal(0, 1.5, (300, n_tok, group * Hkv, D)).astype(np.float32)
    got = ctx.kv_attention(p.cache, cu(q), p.table, p.lens_t, D ** -0.5, out=torch.full(q.shape, float("nan"), device="cuda"))
    ctx.synchronize()
    f = [a.cpu().numpy() for a in p.f]
    keys, values = [], []
    for s, n in enumerate(lens):
        at = (p.table_np[s, np.arange(n) // 16], slice(None), np.arange(n) % 16)
        for which, rows in ((0, keys), (1, values)):
            x = f[which][at].astype(np.float64)
            rows.append(x * np.repeat(f[2 + which][at].astype(np.float64), 32, -1) if qname == "Q8_0" else x)
    want, tol = ref.attention(q, keys, values, lens, D ** -0.5)
    assert (np.abs(got.cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("n_seq", [3, 300])
@pytest.mark.parametrize("one", [0, 1, 4500])
def test_a_batch_of_empty_places(b200, ctx, n_seq, one):
    """Nothing to attend to but one sequence's positions, or nothing at all: zeros for every other row."""
    import torch

    lens = [0] * n_seq
    lens[1] = one
    p = Pool(b200, ctx, b200.F16, 3, 64, 16, lens, seed=24, width=300)
    if one:
        row = p.rng.normal(0, 1, (2, 1, one, 3, 64)).astype(np.float32)
        ctx.kv_write(p.cache, cu(row[0]), cu(row[1]), cu(p.table_np[1:2]), cu(np.array([one], np.int32)))
    q = p.rng.normal(0, 1.5, (n_seq, 1, 6, 64)).astype(np.float32)
    got = ctx.kv_attention(p.cache, cu(q), p.table, p.lens_t, 0.125, out=torch.full(q.shape, float("nan"), device="cuda"))
    ctx.synchronize()
    got = got.cpu().numpy()
    assert not got[[s for s in range(n_seq) if lens[s] == 0]].any()
    if one:
        k, v = p.rows(1)
        want, tol = ref.attention(q[1:2], [k], [v], [one], 0.125)
        assert (np.abs(got[1:2] - want) <= tol).all()


@pytest.mark.parametrize("qname", ["F16", "Q8_0"])
@pytest.mark.parametrize("width", [1, 2, 300])
def test_attention_whatever_the_tables_width(b200, ctx, qname, width):
    """The table's width bounds the lengths, not what is computed: a wide table of short sequences, an exactly full one."""
    Pool(b200, ctx, getattr(b200, qname), 2, 128, 16, [16 * min(width, 2), 3], seed=7, width=width).fill().check_attention(4, 1)


@pytest.mark.parametrize("qname", ["F16", "Q8_0"])
def test_attention_with_scores_far_apart(b200, ctx, qname):
    """One position takes everything; large and tiny magnitudes of q; values whose scales differ by 2^20 along the cache."""
    p = Pool(b200, ctx, getattr(b200, qname), 2, 128, 16, [300, 77], seed=8)
    n = 300
    k = p.rng.normal(0, 1, (2, n, 2, 128)).astype(np.float32)
    v = (p.rng.normal(0, 1, (2, n, 2, 128)) * 2.0 ** p.rng.integers(-10, 10, (2, n, 1, 1))).astype(np.float32)
    ctx.kv_write(p.cache, cu(k), cu(v), p.table, p.lens_t)
    for size in (1e-30, 1e-3, 1.0, 30.0):
        p.check_attention(4, 1, q=(p.rng.normal(0, 1, (2, 1, 4, 128)) * size).astype(np.float32))
    p.check_attention(4, 1, scale=1e-6, q=(p.rng.normal(0, 1, (2, 1, 4, 128)) * 1e6).astype(np.float32))
    p.check_attention(4, 1, scale=0.0)
    p.check_attention(4, 1, scale=-0.1)
    q = np.zeros((2, 1, 4, 128), np.float32)
    p.check_attention(4, 1, q=q)  # the mean of the values


@pytest.mark.parametrize("qname", ["F16", "Q8_0"])
@pytest.mark.parametrize("width", [None, 300])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_with_large_equal_scores(b200, ctx, qname, width, sign):
    """Equal scores of 2^20 to 2^31 (the distances between floats go from 1/8 to 256): the mean of the values, whatever they are."""
    n, D = 200, 64
    p = Pool(b200, ctx, getattr(b200, qname), 1, D, 16, [n], seed=25, width=width)
    k = np.full((1, n, 1, D), 127.0, np.float32)  # the scale 1 in Q8_0
    v = p.rng.normal(0, 1, (1, n, 1, D)).astype(np.float32)
    ctx.kv_write(p.cache, cu(k), cu(v), p.table, p.lens_t)
    ctx.synchronize()
    values = p.rows(0)[1][:, 0]
    # weights that are equal have 22 bits each, as have their products with a scale; a sum of 200, a division: below 2^-19
    tol = np.abs(values).mean(0) * 2.0 ** -19
    for power in range(20, 32):
        for part in (1.0, 1.37, 1.999):
            q = np.full((1, 1, 2, D), sign * part * 2.0 ** power / (127 * D), np.float32)
            got = ctx.kv_attention(p.cache, cu(q), p.table, p.lens_t, 1.0).cpu().numpy()[0, 0]
            assert (np.abs(got - values.mean(0)) <= tol).all(), (power, part)


@pytest.mark.parametrize("n_tok", [1, 3])
def test_values_that_a_weight_all_but_leaves_out(b200, ctx, n_tok):
    """In one piece of the cache lie values of 1e6 whose weights are some e^-40 and values of 1e-4 whose weights are most of
    the sum; in another the scales are 0."""
    p = Pool(b200, ctx, b200.Q8_0, 2, 128, 16, [90], seed=22)
    k = p.rng.normal(0, 0.1, (1, 90, 2, 128)).astype(np.float32)
    v = (p.rng.normal(0, 1, (1, 90, 2, 128)) * 1e-4).astype(np.float32)
    k[:, ::7], v[:, ::7] = -1.0, v[:, ::7] * 1e10
    v[:, 30:41] = 0.0
    ctx.kv_write(p.cache, cu(k), cu(v), p.table, p.lens_t)
    q = np.ones((1, n_tok, 4, 128), np.float32)
    p.check_attention(4, n_tok, scale=0.3125, q=q)  # scores of -40 beside +-0.35


def lay_out(pool, s, which, numbers, scales):
    """Sequence s's rows of a Q8_0 pool as they are given: whole numbers [n][Hkv][D] and scales [n][Hkv][D / 32]."""
    import torch

    pos = np.arange(numbers.shape[0])
    page, slot = (torch.from_numpy(x).cuda() for x in (pool.table_np[s, pos // pool.page].astype(np.int64), pos % pool.page))
    pool.f[which][page, :, slot] = cu(numbers.astype(np.int8))
    pool.f[2 + which][page, :, slot] = cu(scales.astype(np.float16))


@pytest.mark.parametrize("S,width", [(450, None), (450, 300), (1, None), (1, 300)])  # items of their own, or shared; by items, by positions
@pytest.mark.parametrize("least,spread", [(2.0 ** -14, 0), (2.0 ** -13, 0), (2.0 ** -11, 0), (2.0 ** -14, 14), (2.0 ** -13, 13), (2.0 ** -11, 11)])
@pytest.mark.parametrize("n,first", [(40, 3), (900, 500), (4700, 3), (4700, 2600)])
@pytest.mark.parametrize("D,group", [(64, 2), (64, 12), (96, 2), (96, 9), (128, 2), (128, 16), (256, 2)])
def test_a_tail_behind_one_position(b200, ctx, D, group, n, first, least, spread, S, width):
    """One position takes all but e^-17 to e^-22 of the weights, and in the first block its values are 0: there the many small
    weights are all there is. The values' scales are all the same, or go from there to 1. (All sequences are the same one, so
    many that a warp takes a long run of its positions.)"""
    rng = np.random.default_rng(n + D)
    p = Pool(b200, ctx, b200.Q8_0, 1, D, 16, [n], seed=n, width=width)
    blocks = D // 32
    k, kd = np.full((n, 1, D), -127), np.zeros((n, 1, blocks))
    kd[:] = rng.uniform(17, 22, (n, 1, 1)) / (127 * D)  # q is 1 in every dimension: scores of -17 to -22 beside 0
    k[first], kd[first] = 0, 1.0
    v = rng.integers(-127, 128, (n, 1, D))
    vd = least * 2.0 ** (rng.uniform(0, spread, (n, 1, blocks)))
    beside = slice(first, first + 1) if n < 100 else slice(first // 64 * 64, first // 64 * 64 + 64)
    v[beside, 0, :32] = 0  # those that are taken at a time with the first one, too, where there are others
    lay_out(p, 0, 0, k, kd)
    lay_out(p, 0, 1, v, vd)
    q = np.ones((S, 1, group, D), np.float32)
    got = ctx.kv_attention(p.cache, cu(q), p.table.repeat(S, 1), p.lens_t.repeat(S), 1.0).cpu().numpy()[:, 0]
    ctx.synchronize()
    kk, vv = p.rows(0)
    score = kk[:, 0].sum(-1)
    w = np.exp(score - score.max())
    w /= w.sum()
    want, size = w @ vv[:, 0], w @ np.abs(vv[:, 0])
    # A score is D / 32 exact blocks added up and two products more, each off by at most half a unit of 32 (2^-19), as are the
    # two differences of base-2 logarithms that its weight is the exponential of: an error of delta in every score changes a
    # weight by at most exp(2 delta) - 1. The weight meets up to four exponentials (2^-22 each), enters with 22 bits, as does
    # its product with a scale, and is divided: below 2^-19. A warp takes at most 16 of every 64 positions, each 16 are
    # added once, and up to 34 partial results are joined. F16 holds a weight and its product with a scale (at most 1) to 2^-39
    # each of the largest weight, or twice that, that it is taken with: the first one's for 31 positions where these have
    # values, the tail's for the others.
    delta = (D / 32 + 4) * 2.0 ** -19
    tol = size * (np.expm1(2 * delta) + 2.0 ** -19 + (n / 64 + 34) * 2.0 ** -24)
    tol += 127 * 2.0 ** -38 * np.where((np.arange(D) < 32) & (n > 100), 0, 31) + n * 127 * 2.0 ** -37 * np.exp(-17)
    assert (np.abs(got - want) <= tol).all(), f"off by {np.max(np.abs(got - want) / size):.3g} of the magnitudes, allowed {np.max(tol / size):.3g}"


@pytest.mark.parametrize("width", [None, 300])
def test_attention_does_not_see_what_lies_behind_a_row(b200, ctx, width):
    """Positions that later rows of the call see, but an earlier one does not, hold NaN and infinities: the earlier rows
    come out as if these were not there; the later ones are NaN where the definition is."""
    import torch

    p = Pool(b200, ctx, b200.F16, 2, 128, 16, [50, 17], seed=9, width=width).fill()
    q = p.rng.normal(0, 1, (2, 4, 4, 128)).astype(np.float32)
    clean = ctx.kv_attention(p.cache, cu(q), p.table, p.lens_t, 0.1)
    for which, value in ((0, float("nan")), (1, float("nan")), (1, float("inf")), (0, float("inf"))):
        keep = p.data.clone()
        for s, n in enumerate(p.lens):
            p.f[which][p.table_np[s, (n - 2) // 16], :, (n - 2) % 16] = value  # rows 2 and 3 see it
        got = ctx.kv_attention(p.cache, cu(q), p.table, p.lens_t, 0.1)
        assert torch.equal(got[:, :2], clean[:, :2])
        assert not torch.isfinite(got[:, 2:]).all(-1).any()
        p.data.copy_(keep)
    ctx.synchronize()


@pytest.mark.parametrize("qname", ["F16", "Q8_0"])
@pytest.mark.parametrize("D,H", [(64, 4), (64, 8), (96, 8), (128, 4), (128, 8), (256, 8)])  # eight rows of a key/value head, or sixteen
@pytest.mark.parametrize("width", [None, 300])
def test_rows_before_a_position_that_is_not_finite(b200, ctx, qname, D, H, width):
    """A key or value (in Q8_0: its scale) that only the later half of the call's rows see is NaN or infinite: the earlier
    rows have what they have without it."""
    import torch

    p = Pool(b200, ctx, getattr(b200, qname), 2, D, 16, [50, 17, 135], seed=28, width=width).fill()
    q = p.rng.normal(0, 1, (3, 4, H, D)).astype(np.float32)
    kv = [p.rows(s) for s in range(3)]
    want, tol = ref.attention(q[:, :2], [k[:-2] for k, _ in kv], [v[:-2] for _, v in kv], [n - 2 for n in p.lens], 0.1)
    first = 0 if qname == "F16" else 2
    for which, value in ((0, float("nan")), (0, float("inf")), (1, float("nan")), (1, float("inf"))):
        keep = p.data.clone()
        for s, n in enumerate(p.lens):
            p.f[first + which][p.table_np[s, (n - 2) // 16], :, (n - 2) % 16] = value  # rows 2 and 3 see it
        got = ctx.kv_attention(p.cache, cu(q), p.table, p.lens_t, 0.1)
        assert (np.abs(got[:, :2].cpu().numpy() - want) <= tol).all()
        if which == 1 or np.isnan(value):
            assert not torch.isfinite(got[:, 2:]).all(-1).any()
        p.data.copy_(keep)
    ctx.synchronize()


@pytest.mark.parametrize("D,Hkv,group,page,n_tok,lens", [(64, 2, 2, 16, 1, [300]), (64, 1, 5, 48, 3, [200, 31]), (96, 2, 1, 16, 1, [100, 700]),
                                                         (96, 1, 16, 32, 1, [333]), (128, 1, 4, 16, 4, [260, 5]), (256, 2, 2, 32, 2, [90, 400])])
@pytest.mark.parametrize("width", [None, 300])
def test_value_scales_of_any_size(b200, ctx, D, Hkv, group, page, n_tok, lens, width):
    """Blocks whose scales lie below 2^-14, above 2, in between and across these ends."""
    p = Pool(b200, ctx, b200.Q8_0, Hkv, D, page, lens, seed=29, width=width)
    n = max(lens)
    k = p.rng.normal(0, 1, (len(lens), n, Hkv, D)).astype(np.float32)
    blocks = np.resize([2.0 ** -16, 2.0 ** 12, 1.0, 2.0 ** -7, 2.0 ** 7, 2.0 ** -20], (Hkv * D // 32,)).reshape(Hkv, D // 32).repeat(32, -1)
    v = (p.rng.normal(0, 1, (len(lens), n, Hkv, D)) * 2.0 ** p.rng.integers(-2, 3, (len(lens), n, Hkv, 1)) * blocks).astype(np.float32)
    ctx.kv_write(p.cache, cu(k), cu(v), p.table, p.lens_t)
    p.check_attention(Hkv * group, n_tok)


@pytest.mark.parametrize("qname", ["F16", "Q8_0"])
def test_a_prefix_read_back_for_a_prompts_block(b200, ctx, qname):
    """The rows of one request taken out as F16 and attended to by FLASH_ATTN: the 30 newest of 77 positions, of which the 16
    newest are what kv_attention gives for them."""
    import torch

    n, n_q, H, Hkv, D, scale = 77, 30, 4, 2, 64, 0.125
    p = Pool(b200, ctx, getattr(b200, qname), Hkv, D, 16, [n], seed=30).fill()
    k, v = ctx.kv_read(p.cache, p.table, p.lens_t, n_tok=n, dtype=torch.float16)
    q = p.rng.normal(0, 1, (n_q, H, D)).astype(np.float16).astype(np.float32)  # FLASH_ATTN rounds q to F16
    mask = np.where(np.arange(n)[None] <= n - n_q + np.arange(n_q)[:, None], 0.0, -np.inf).astype(np.float16)
    out, qd, md = torch.full((n_q, H, D), float("nan"), device="cuda"), cu(q), cu(mask)
    g = b200.Graph(ctx)
    g.add(b200.OP_FLASH_ATTN, out, src=[g.add(t=t) for t in (qd.permute(1, 0, 2), k[0].permute(1, 0, 2), v[0].permute(1, 0, 2), md)],
          params=[g.fbits(scale)])
    g.compute()
    newest = ctx.kv_attention(p.cache, qd[None, -16:].contiguous(), p.table, p.lens_t, scale)
    ctx.synchronize()
    kk, vv = (x[0].cpu().numpy().astype(np.float64) for x in (k, v))
    for which, x in enumerate(p.rows(0)):  # the rows are the cache's, rounded once
        assert np.array_equal((kk, vv)[which], x.astype(np.float32).astype(np.float16).astype(np.float64))
    s = np.einsum("qhd,jhd->qhj", q.astype(np.float64), kk.repeat(H // Hkv, 1)) * scale + mask[:, None].astype(np.float64)
    w = np.exp(s - s.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    want, size = (np.einsum("qhj,jhd->qhd", w, x.repeat(H // Hkv, 1)) for x in (vv, np.abs(vv)))
    # a score is rounded twice, its difference to the maximum and its exponential once, a product with a value and the result once
    delta = 4 * 2.0 ** -24 * np.abs(np.where(np.isfinite(s), s, 0)).max()
    assert (np.abs(out.cpu().numpy() - want) <= size * (np.expm1(2 * delta) + 2.0 ** -22)).all()
    got = newest[0].cpu().numpy()
    want, tol = ref.attention(q[None, -16:], [p.rows(0)[0]], [p.rows(0)[1]], [n], scale)
    assert (np.abs(got - want[0]) <= tol[0]).all()


def test_non_finite_queries_stay_in_their_rows(b200, ctx):
    import torch

    p = Pool(b200, ctx, b200.F16, 2, 128, 16, [50], seed=10).fill()
    q = p.rng.normal(0, 1, (1, 2, 4, 128)).astype(np.float32)
    clean = ctx.kv_attention(p.cache, cu(q), p.table, p.lens_t, 0.1)
    for value in (np.nan, np.inf, -np.inf):
        q2 = q.copy()
        q2[0, 1, 2, 5] = value
        got = ctx.kv_attention(p.cache, cu(q2), p.table, p.lens_t, 0.1)
        same = torch.ones(1, 2, 4, dtype=torch.bool, device="cuda")
        same[0, 1, 2] = False
        assert torch.equal(got[same], clean[same]) and torch.isnan(got[0, 1, 2]).all()


@pytest.mark.parametrize("longest", [3000, 7000])
def test_attention_gives_the_same_bits_every_time(b200, ctx, longest):
    import torch

    p = Pool(b200, ctx, b200.Q8_0, 2, 128, 16, [longest, 1, 700, 2999], seed=11).fill()
    q = cu(p.rng.normal(0, 1, (4, 2, 8, 128)).astype(np.float32))
    first = ctx.kv_attention(p.cache, q, p.table, p.lens_t, 0.1)
    for _ in range(5):
        assert torch.equal(first, ctx.kv_attention(p.cache, q, p.table, p.lens_t, 0.1))


def test_places_past_4_gib(b200, ctx):
    """Pages whose byte offsets pass 2^31 and 2^32."""
    import torch

    Hkv, D, page, n_pages = 8, 256, 4096, 290  # 16 MiB a page and array: 4.5 GiB of keys
    cache = ctx.kv_cache(b200.F16, Hkv, D, page, n_pages)
    rng = np.random.default_rng(12)
    n = 40
    k, v = (rng.normal(0, 1, (2, n, Hkv, D)).astype(np.float32) for _ in range(2))
    table, lens = cu(np.array([[n_pages - 1], [130]], np.int32)), cu(np.array([n, n], np.int32))
    ctx.kv_write(cache, cu(k), cu(v), table, lens)
    kk, vv = ctx.kv_read(cache, table, lens, n_tok=n)
    assert np.array_equal(kk.cpu().numpy(), k.astype(np.float16).astype(np.float32))
    assert np.array_equal(vv.cpu().numpy(), v.astype(np.float16).astype(np.float32))
    q = rng.normal(0, 1, (2, 1, 8, D)).astype(np.float32)
    got = ctx.kv_attention(cache, cu(q), table, lens, 0.0625).cpu().numpy()
    want, tol = ref.attention(q, k.astype(np.float16), v.astype(np.float16), [n, n], 0.0625)
    assert (np.abs(got - want) <= tol).all()
    cache.close()
    ctx.synchronize()
    torch.cuda.empty_cache()


# ---- streams and graphs ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("lens", [[4000, 3500], [6000, 5500]])  # by items; by positions, with a workspace
def test_calls_run_on_torchs_current_stream(b200, ctx, lens):
    """Two streams at once, each with its own sequences of one pool: no call waits for or reads the other's workspace."""
    import torch

    p = Pool(b200, ctx, b200.F16, 2, 128, 16, lens, seed=13).fill()
    q = cu(p.rng.normal(0, 1, (2, 1, 8, 128)).astype(np.float32))
    want = [ctx.kv_attention(p.cache, q[i:i + 1], p.table[i:i + 1], p.lens_t[i:i + 1], 0.1) for i in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ctx.kv_attention(p.cache, q[i:i + 1], p.table[i:i + 1], p.lens_t[i:i + 1], 0.1))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, want[i]) for x in got[i])
    # the context's own stream (a NULL stream in the C call)
    out = torch.zeros_like(want[0])
    size = ctx.L.b200_kv_attention_workspace(ctx.h, p.cache.ref, p.width, 1, 1, 8)
    ws = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.check(ctx.L.b200_kv_attention(ctx.h, None, p.cache.ref, p.table.data_ptr(), p.width, p.lens_t.data_ptr(), 1, 1, 8, q.data_ptr(), 1024, 0.1,
                                      out.data_ptr(), ws.data_ptr(), size))
    ctx.synchronize()
    assert torch.equal(out, want[0])


@pytest.mark.parametrize("others", [1, 2])
def test_synchronize_waits_for_the_streams_that_calls_ran_on(b200, ctx, others):
    """Calls on side streams, checked outside of these: their work is done and their errors are raised, once."""
    import torch

    p = Pool(b200, ctx, b200.F16, 1, 64, 16, [20], seed=27).fill()
    q, bad = torch.ones(1, 1, 1, 64, device="cuda"), cu(np.array([-1], np.int32))
    outs = [torch.ones(1, 1, 1, 64, device="cuda") for _ in range(others)]
    ctx.synchronize()
    for rep in range(3):
        streams = [torch.cuda.Stream() for _ in range(others)]
        for st, out in zip(streams, outs):
            out.fill_(1.0)
            torch.cuda.synchronize()
            with torch.cuda.stream(st):
                torch.cuda._sleep(10_000_000)  # some 5 ms
                ctx.kv_attention(p.cache, q, p.table, bad, 1.0, out=out)
        with pytest.raises(b200.B200Error, match="kv cache"):
            ctx.synchronize()
        assert all(st.query() for st in streams)
        assert not any(out.any() for out in outs)
        ctx.synchronize()


def test_the_first_call_of_a_context_may_be_captured(b200):
    import torch

    for lens in ([300, 5], [6000, 5]):  # by items, by positions
        fresh = b200.Context(0)
        p = Pool(b200, fresh, b200.F16, 2, 64, 16, lens, seed=21)
        n = max(lens)
        k, v = (torch.randn(2, n, 2, 64, device="cuda") for _ in range(2))
        q, out = torch.randn(2, 1, 4, 64, device="cuda"), torch.zeros(2, 1, 4, 64, device="cuda")
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            fresh.kv_write(p.cache, k, v, p.table, p.lens_t)
            fresh.kv_attention(p.cache, q, p.table, p.lens_t, 0.2, out=out)
        graph.replay()
        assert torch.equal(out, fresh.kv_attention(p.cache, q, p.table, p.lens_t, 0.2)) and out.any()
        fresh.synchronize()
        del graph
        fresh.close()


@pytest.mark.parametrize("longest", [700, 5000])
@pytest.mark.parametrize("qname", ["F16", "Q8_0"])
def test_a_captured_step_replays_with_new_rows_and_lengths(b200, ctx, qname, longest):
    """Write and attention captured once, replayed while the sequences grow over page ends; two graphs replayed at once."""
    import torch

    page, steps = 16, 40
    lens0 = [1, 10, longest]
    p = Pool(b200, ctx, getattr(b200, qname), 2, 64, page, [n + steps for n in lens0], seed=14).fill()
    graphs = []
    for _ in range(2):
        st = dict(k=torch.zeros(3, 1, 2, 64, device="cuda"), v=torch.zeros(3, 1, 2, 64, device="cuda"), q=torch.zeros(3, 1, 4, 64, device="cuda"),
                  lens=cu(np.array(lens0, np.int32)), out=torch.zeros(3, 1, 4, 64, device="cuda"), graph=torch.cuda.CUDAGraph())
        ctx.kv_attention(p.cache, st["q"], p.table, st["lens"], 0.2, out=st["out"])  # warm
        torch.cuda.synchronize()
        with torch.cuda.graph(st["graph"]):
            ctx.kv_write(p.cache, st["k"], st["v"], p.table, st["lens"])
            ctx.kv_attention(p.cache, st["q"], p.table, st["lens"], 0.2, out=st["out"])
        graphs.append(st)
    a, b = graphs
    for step in range(steps):
        for name in ("k", "v", "q"):
            a[name].copy_(cu(p.rng.normal(0, 1, a[name].shape).astype(np.float32)))
            b[name].copy_(a[name])
        a["graph"].replay()
        eager = ctx.kv_attention(p.cache, a["q"], p.table, a["lens"], 0.2)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            b["graph"].replay()  # the same rows to the same places, at the same time as the first graph
        a["graph"].replay()
        torch.cuda.synchronize()
        assert torch.equal(a["out"], eager) and torch.equal(b["out"], eager)
        if step % 13 == 0:
            p.lens = [n + step for n in lens0]
            kv = [p.rows(s) for s in range(3)]
            want, tol = ref.attention(a["q"].cpu().numpy(), [x for x, _ in kv], [x for _, x in kv], p.lens, 0.2)
            assert (np.abs(eager.cpu().numpy() - want) <= tol).all()
        a["lens"] += 1
        b["lens"] += 1
    ctx.synchronize()
