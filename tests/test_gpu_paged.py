"""The paged cache: the append with rotation, and attention of one new token per sequence,
against plain forms in 64 bits.

Tolerances.  u is half a step of the output's type (2^-8 bf16, 2^-11 f16).  An appended
value is one rounding of an f32 expression of three operations: u |y| + 2^-22 (|a| + |b|).
An attention output o = sum w_j v_j carries its own rounding (u |o|), the rounding of each
p_j to 16 bits (u sum w_j |v_j|), the f32 error of the scores, which moves each p_j by at
most e = 2^-24 (head_dim + 4) * max |q||k| scale + 2^-21 relative (and the sum as much), the f32
sums over n keys (n 2^-24) and, for f16, the 2^-25 that a p below 2^-14 may be off, the
largest p being at least one.  Over Q8_0 the products are of integers: a query value is a
multiple of amax / 32512 of its block of 32, so off by amax / 65024, which moves a score by
scale * sum |k_d| amax / 65024 at most (e grows by twice that); and p times a value's scale is
a multiple of 1 / 65534 of the largest p times the largest scale among 32 keys (from a multiple
of 32 on), so each of the 32 adds at most 127 / 131068 of that product to the error."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def ids(ncm):
    return {"f16": ncm.F16, "bf16": ncm.BF16, "q8_0": ncm.Q8_0, "f32": ncm.F32}


class Cache:
    """A cache whose unused places hold NaN (scales NaN, int8 127), and its page table."""

    def __init__(self, ncm, kind, kvh, hd, page, totals, seed, spare=3, interleaved=False, width=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        need = [-(-max(n, 0) // page) for n in totals]
        self.width = width or max(1, max(need))
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(totals), self.width), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.kind, self.kvh, self.hd, self.page, self.totals, self.g = kind, kvh, hd, page, totals, g
        shape = (self.pages, kvh, page, hd)
        self.ks = self.vs = None
        stride = 0
        if kind == "q8_0":
            self.k, self.v = (torch.full(shape, 127, dtype=torch.int8, device="cuda") for _ in range(2))
            self.ks, self.vs = (torch.full(shape[:3] + (hd // 32,), float("nan"), dtype=torch.float16, device="cuda")
                                for _ in range(2))
        elif interleaved:   # K and V of a page side by side
            both = torch.full((self.pages, 2) + shape[1:], float("nan"), dtype=DT[kind], device="cuda")
            self.k, self.v, stride = both[:, 0], both[:, 1], 2 * kvh * page * hd
        else:
            self.k, self.v = (torch.full(shape, float("nan"), dtype=DT[kind], device="cuda") for _ in range(2))
        q8 = kind == "q8_0"
        self.kv = ncm.PagedKV(ids(ncm)[kind], self.k.data_ptr(), self.v.data_ptr(), self.pages, page, kvh, hd,
                              self.ks.data_ptr() if q8 else 0, self.vs.data_ptr() if q8 else 0, stride)

    def fill(self, scale_k=1.0):
        """Random rows for every sequence."""
        for i, n in enumerate(self.totals):
            if n <= 0:
                continue
            pos = torch.arange(n, device="cuda")
            pg, off = self.table[i].long()[pos // self.page], pos % self.page
            for x, s, f in ((self.k, self.ks, scale_k), (self.v, self.vs, 1.0)):
                if self.kind == "q8_0":
                    x[pg, :, off] = torch.randint(-127, 128, (n, self.kvh, self.hd), generator=self.g, device="cuda", dtype=torch.int8)
                    s[pg, :, off] = (torch.rand((n, self.kvh, self.hd // 32), generator=self.g, device="cuda") * 0.02 * f + 1e-4).half()
                else:
                    x[pg, :, off] = (torch.randn((n, self.kvh, self.hd), generator=self.g, device="cuda") * f).to(x.dtype)
        return self

    def rows(self, which, i, n):
        """The values of sequence i's first n rows in 64 bits, [n, kvh, hd]."""
        x, s = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        pos = torch.arange(n, device="cuda")
        pg, off = self.table[i].long()[pos // self.page], pos % self.page
        y = x[pg, :, off].double()
        if which == "v_scales":
            return s[pg, :, off] if s is not None else None
        return y * s[pg, :, off].double().repeat_interleave(32, -1) if self.kind == "q8_0" else y


def attend64(q, k, v, scale, qkind, hd, v_scales=None):
    """One query [heads, hd] over [n, kvh, hd] in 64 bits: the output and its tolerance.
    v_scales [n, kvh, hd / 32]: of a Q8_0 cache."""
    heads, g = q.shape[0], q.shape[0] // k.shape[1]
    if k.shape[0] == 0:
        return torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = torch.einsum("hd,nhd->hn", q.double(), k) * scale
    top = (torch.einsum("hd,nhd->hn", q.double().abs(), k.abs()) * scale).amax(-1)[:, None]
    w = torch.softmax(s, -1)
    o, a = torch.einsum("hn,nhd->hd", w, v), torch.einsum("hn,nhd->hd", w, v.abs())
    n, u = k.shape[0], U[qkind]
    e = 2 * (2.0 ** -24 * (hd + 4) * top + 2.0 ** -21) + n * 2.0 ** -24
    small = 2.0 ** -25 * (1 + n * v.abs().amax()) if qkind == "f16" else 0.0
    if v_scales is not None:
        step = q.double().abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1) / 65024
        e = e + 2 * (torch.einsum("hd,nhd->hn", step, k.abs()) * scale).amax(-1)[:, None]
        pad = -n % 32
        wu = torch.nn.functional.pad(w, (0, pad)).unflatten(-1, (-1, 32)).amax(-1)                               # [h, units]
        su = torch.nn.functional.pad(v_scales.double(), (0, 0, 0, 0, 0, pad)).unflatten(0, (-1, 32)).amax(1)    # [units, kvh, hd / 32]
        su = su.repeat_interleave(g, 1).repeat_interleave(32, -1)
        small = small + torch.einsum("hu,uhd->hd", wu, su) * (32 * 127 / 131068)
    return o, u * o.abs() + (u + e) * a * (1 + u) + small


def attend(ncm, c, q, lengths, heads, qkind, out=None, scale=0.0, err=None, space=None, stream=0, q_stride=0, out_stride=0):
    out = torch.full_like(q, float("nan")) if out is None else out
    space = torch.zeros(ncm.paged_attention_workspace(heads, c.kvh, c.hd), dtype=torch.uint8, device="cuda") if space is None else space
    ncm.paged_attention(out.data_ptr(), q.data_ptr(), c.kv, ids(ncm)[qkind], lengths.numel(), heads, lengths.data_ptr(),
                        c.table.data_ptr(), c.width, space.data_ptr(), space.numel(), scale=scale, q_stride=q_stride,
                        out_stride=out_stride, err_ptr=err.data_ptr() if err is not None else 0, stream=stream)
    return out


def check(c, q, out, lengths, qkind, scale=None):
    scale = c.hd ** -0.5 if scale is None else scale
    for i, n in enumerate(lengths):
        ref, tol = attend64(q[i], c.rows("k", i, max(n, 0)), c.rows("v", i, max(n, 0)), scale, qkind, c.hd, c.rows("v_scales", i, max(n, 0)))
        off = (out[i].double() - ref).abs()
        assert bool((off <= tol).all()), (i, n, float((off - tol).max()), float(off.max()))


def int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


RAGGED = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300, 1000]


@pytest.mark.parametrize("kind,qkind", [("f16", "f16"), ("bf16", "bf16"), ("q8_0", "f16"), ("q8_0", "bf16")])
@pytest.mark.parametrize("heads,kvh,hd,page", [(8, 2, 64, 16), (8, 2, 128, 8), (6, 2, 128, 64), (16, 2, 128, 256),
                                               (4, 4, 64, 32), (12, 1, 128, 16), (40, 2, 64, 8), (64, 2, 128, 32)])
def test_attention_ragged(ncm, cuda, kind, qkind, heads, kvh, hd, page):
    c = Cache(ncm, kind, kvh, hd, page, RAGGED, seed=heads + hd).fill()
    q = torch.randn((len(RAGGED), heads, hd), generator=c.g, device="cuda").to(DT[qkind])
    out = attend(ncm, c, q, int32(RAGGED), heads, qkind)
    assert bool((out[0] == 0).all())
    check(c, q, out, RAGGED, qkind)


@pytest.mark.parametrize("kind,qkind", [("f16", "f16"), ("bf16", "bf16"), ("q8_0", "f16")])
@pytest.mark.parametrize("lengths,heads,kvh,hd,page", [([1], 4, 1, 128, 16), ([1], 32, 8, 64, 16), ([70001], 8, 1, 128, 64),
                                                       ([30011], 16, 2, 64, 16), ([5000, 1, 9000], 8, 2, 128, 32),
                                                       ([0, 0, 0], 8, 2, 64, 8), ([4096, 0, 4095, 4097], 32, 8, 128, 128)])
def test_attention_split(ncm, cuda, kind, qkind, lengths, heads, kvh, hd, page):
    """Few long sequences: the keys of a head are shared out over many CTAs and joined."""
    c = Cache(ncm, kind, kvh, hd, page, lengths, seed=sum(lengths) % 1000).fill()
    q = (torch.randn((len(lengths), heads, hd), generator=c.g, device="cuda") * 2).to(DT[qkind])
    space = torch.zeros(ncm.paged_attention_workspace(heads, kvh, hd), dtype=torch.uint8, device="cuda")
    out = attend(ncm, c, q, int32(lengths), heads, qkind, space=space)
    check(c, q, out, lengths, qkind)
    assert int(space[:4096].sum()) == 0   # counters are left at zero
    for _ in range(3):   # and the same bits come out whoever finishes last
        assert torch.equal(attend(ncm, c, q, int32(lengths), heads, qkind, space=space), out)


def test_attention_peaked_and_scaled(ncm, cuda):
    """Scores that grow along the sequence by hundreds: the running maximum has to follow."""
    n, heads, kvh, hd = 3000, 8, 2, 128
    c = Cache(ncm, "bf16", kvh, hd, 16, [n], seed=5).fill()
    pos = torch.arange(n, device="cuda")
    c.k[c.table[0].long()[pos // 16], :, pos % 16] = (torch.linspace(-4, 4, n, device="cuda")[:, None, None]
                                                    * torch.ones(kvh, hd, device="cuda")).bfloat16()
    q = torch.ones((1, heads, hd), device="cuda").bfloat16()
    q[:, 1::2] = -1.0
    for scale in (0.05, 1.0):
        out = attend(ncm, c, q, int32([n]), heads, "bf16", scale=scale)
        check(c, q, out, [n], "bf16", scale)


def test_attention_strides_interleaved_pages_and_rows_behind(ncm, cuda):
    """q as a slice of a wider row, out rows apart, K and V in one allocation; neither the rows
    between nor the rows behind the last sequence change."""
    heads, kvh, hd, lengths = 8, 2, 128, [5, 77, 0, 40]
    c = Cache(ncm, "f16", kvh, hd, 16, lengths, seed=9, interleaved=True).fill()
    wide = torch.randn((4, heads + 2 * kvh, hd), generator=c.g, device="cuda").half()
    out = torch.full((7, heads + 3, hd), 7.0, dtype=torch.float16, device="cuda")
    attend(ncm, c, wide, int32(lengths), heads, "f16", out=out, q_stride=(heads + 2 * kvh) * hd, out_stride=(heads + 3) * hd)
    check(c, wide[:, :heads], out[:4, :heads], lengths, "f16")
    assert bool((out[4:] == 7).all()) and bool((out[:, heads:] == 7).all())


def test_attention_shared_pages_are_one_sequence_many_rows(ncm, cuda):
    """Speculative rows: the same pages, lengths one apart."""
    heads, kvh, hd, n = 8, 2, 64, 500
    c = Cache(ncm, "bf16", kvh, hd, 32, [n], seed=2).fill()
    c.table = c.table.expand(6, -1).contiguous()
    lengths = [n - 5 + i for i in range(6)]
    q = torch.randn((6, heads, hd), generator=c.g, device="cuda").bfloat16()
    check(c, q, attend(ncm, c, q, int32(lengths), heads, "bf16"), lengths, "bf16")


def test_attention_many_sequences(ncm, cuda):
    """More sequences than one launch takes."""
    rng = np.random.default_rng(4)
    lengths = [int(x) for x in rng.integers(0, 40, 2300)]
    c = Cache(ncm, "f16", 1, 64, 16, [40], seed=3).fill()
    c.table = c.table.expand(2300, -1).contiguous()
    q = torch.randn((2300, 4, 64), generator=c.g, device="cuda").half()
    out = attend(ncm, c, q, int32(lengths), 4, "f16")
    k, v = c.rows("k", 0, 40), c.rows("v", 0, 40)
    for i in list(range(0, 2300, 97)) + [2047, 2048, 2299]:
        ref, tol = attend64(q[i], k[:lengths[i]], v[:lengths[i]], 0.125, "f16", 64)
        assert bool(((out[i].double() - ref).abs() <= tol).all()), i


def test_attention_far_pages(ncm, cuda):
    """Pages whose elements lie past 2^31."""
    kvh, hd, page, n = 8, 128, 64, 100
    pages = 2 ** 31 // (kvh * page * hd) + 40
    k = torch.empty((pages, kvh, page, hd), dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    c = Cache(ncm, "f16", kvh, hd, page, [n, n], seed=1)
    c.k, c.v, c.pages = k, v, pages
    c.table = int32([[pages - 1, 3], [7, pages - 2]])
    c.kv = ncm.PagedKV(ncm.F16, k.data_ptr(), v.data_ptr(), pages, page, kvh, hd)
    c.fill()
    q = torch.randn((2, 16, hd), generator=c.g, device="cuda").half()
    check(c, q, attend(ncm, c, q, int32([n, n]), 16, "f16"), [n, n], "f16")


def test_attention_bad_lengths_and_pages_are_flagged(ncm, cuda):
    """A length past the table is cut, a bad page id reads as zeros; the others are right."""
    heads, kvh, hd, lengths = 8, 2, 64, [30, 64, -5, 50]
    c = Cache(ncm, "f16", kvh, hd, 16, [30, 64, 0, 50], seed=6).fill()
    err = int32([0])
    q = torch.randn((4, heads, hd), generator=c.g, device="cuda").half()
    out = attend(ncm, c, q, int32(lengths), heads, "f16", err=err)
    check(c, q, out, lengths, "f16")
    assert err.item() == 0
    out = attend(ncm, c, q, int32([30, 1000, 0, 50]), heads, "f16", err=err)
    check(c, q, out, [30, 64, 0, 50], "f16")
    assert err.item() == ncm.DEVICE_BAD_ARG
    for page in (-1, -2 ** 31, c.pages, 2 ** 31 - 1):
        err.zero_()
        bad = c.table.clone()
        bad[1, 1] = page
        good, c.table = c.table, bad
        out = attend(ncm, c, q, int32([30, 64, 0, 50]), heads, "f16", err=err)
        c.table = good
        for i in (0, 2, 3):
            ref, tol = attend64(q[i], c.rows("k", i, lengths[i] if i != 2 else 0), c.rows("v", i, lengths[i] if i != 2 else 0), 0.125, "f16", 64)
            assert bool(((out[i].double() - ref).abs() <= tol).all())
        assert err.item() == ncm.DEVICE_BAD_ARG and bool(out[1].isfinite().all())


def test_attention_nan_in_a_key_stays_in_its_sequence(ncm, cuda):
    heads, kvh, hd, lengths = 4, 1, 64, [40, 70, 33]
    c = Cache(ncm, "bf16", kvh, hd, 16, lengths, seed=8).fill()
    c.k[c.table[1, 2].item(), 0, 3, 5] = float("nan")
    q = torch.randn((3, heads, hd), generator=c.g, device="cuda").bfloat16()
    out = attend(ncm, c, q, int32(lengths), heads, "bf16")
    assert bool(out[1].isnan().all())
    for i in (0, 2):
        ref, tol = attend64(q[i], c.rows("k", i, lengths[i]), c.rows("v", i, lengths[i]), 0.125, "bf16", 64)
        assert bool(((out[i].double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("n", [5, 40, 3000, 40000])
def test_attention_with_all_scores_minus_infinity(ncm, cuda, n):
    """Keys of -infinity in one sequence: its rows are zeros, as if it had no keys; whole segments,
    parts joined in one CTA, and parts joined over few and many."""
    heads, kvh, hd = 8, 2, 64
    c = Cache(ncm, "bf16", kvh, hd, 64, [n, 50], seed=13).fill()
    pages = c.table[0, :-(-n // 64)].long()
    c.k[pages] = float("-inf")
    q = torch.rand((2, heads, hd), generator=c.g, device="cuda").bfloat16() + 1
    out = attend(ncm, c, q, int32([n, 50]), heads, "bf16")
    assert bool((out[0] == 0).all())
    ref, tol = attend64(q[1], c.rows("k", 1, 50), c.rows("v", 1, 50), 0.125, "bf16", hd)
    assert bool(((out[1].double() - ref).abs() <= tol).all())


def test_attention_in_graphs_and_streams(ncm, cuda):
    """Two captured graphs that share a workspace, replayed in turn with new lengths and inputs."""
    heads, kvh, hd = 16, 2, 128
    c = Cache(ncm, "bf16", kvh, hd, 16, [9000, 4000], seed=12).fill()
    lengths, q = int32([9000, 4000]), torch.randn((2, heads, hd), generator=c.g, device="cuda").bfloat16()
    space = torch.zeros(ncm.paged_attention_workspace(heads, kvh, hd), dtype=torch.uint8, device="cuda")
    outs, graphs, s = [torch.zeros_like(q) for _ in range(2)], [], torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for out in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            attend(ncm, c, q, lengths, heads, "bf16", out=out, space=space, stream=s.cuda_stream)
        graphs.append(g)
    for n in ([9000, 4000], [1, 0], [8191, 33]):
        lengths.copy_(int32(n))
        q.copy_(torch.randn(q.shape, generator=c.g, device="cuda"))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        check(c, q, outs[0], n, "bf16")
        assert torch.equal(outs[0], outs[1])


# ---------------------------------------------------------------- append
def rope_table(n, half, hd, seed=0):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 500000.0 ** (-torch.arange(half, dtype=torch.float64) * 2 / hd)
    return torch.stack([a.sin(), a.cos()], -1).float().cuda()


def rotated64(x, sc, style, half):
    """x [T, H, hd] (64 bits), sc [T, half, 2]: the rotated rows, and |a| + |b| of each value."""
    y, m = x.clone(), x.abs().clone()
    s, c = sc[:, None, :, 0].double(), sc[:, None, :, 1].double()
    if style == "pairs":
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, a * s + b * c
        m[..., 0:2 * half:2] = m[..., 1:2 * half:2] = a.abs() + b.abs()
    else:
        a, b = x[..., :half], x[..., half:]
        y = torch.cat([a * c - b * s, a * s + b * c], -1)
        m = torch.cat([a.abs() + b.abs()] * 2, -1)
    return y, m


def rotated32(x, sc, style, half):
    """The same in f32 with every product and sum rounded, as numpy rounds them."""
    x, sc = x.float().cpu().numpy(), sc.cpu().numpy()
    s, c, y = sc[:, None, :, 0], sc[:, None, :, 1], x.copy()
    if style == "pairs":
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :half], x[..., half:]
        y[..., :half], y[..., half:] = a * c - b * s, a * s + b * c
    return y


def quantised(y):
    """Q8_0 of f32 rows by the rule of the header: int8 values and f16 scales (bits)."""
    blk = y.reshape(y.shape[:-1] + (-1, 32))
    sc = (np.abs(blk).max(-1) * (np.float32(1) / np.float32(127))).astype(np.float32)
    with np.errstate(divide="ignore", over="ignore"):
        inv = np.where(sc > 0, np.float32(1) / sc, np.float32(0)).astype(np.float32)
    t = (blk * inv[..., None]).astype(np.float32).astype(np.float64)
    q = np.clip(np.sign(t) * np.floor(np.abs(t) + 0.5), -127, 127).astype(np.int8)
    h = sc.astype(np.float16)
    up = h.astype(np.float32) > sc
    bits = h.view(np.uint16) - up.astype(np.uint16)
    return q.reshape(y.shape), bits


def append(ncm, c, rows, heads, counts, totals, qkind, inkind, rope, style, half, cu=True, err=None, out=None, stream=0):
    tokens = rows.shape[0]
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    out = torch.full((tokens, heads, c.hd), 9.0, dtype=DT[qkind], device="cuda") if out is None else out
    es, stride = rows.element_size(), rows.shape[1] * c.hd
    keep = (int32(at), int32(totals))
    ncm.paged_append(c.kv, ids(ncm)[inkind], rows.data_ptr(), rows.data_ptr() + es * heads * c.hd,
                     rows.data_ptr() + es * (heads + c.kvh) * c.hd, out.data_ptr(), ids(ncm)[qkind], tokens, heads,
                     len(counts), keep[0].data_ptr() if cu else 0, keep[1].data_ptr(), c.table.data_ptr(), c.width,
                     rope_ptr=rope.data_ptr() if rope is not None else 0, rope_len=rope.shape[0] if rope is not None else 0,
                     rope_half=half, rope_style=ncm.ROPE_PAIRS if style == "pairs" else ncm.ROPE_HALVES, q_stride=stride,
                     k_stride=stride, v_stride=stride, err_ptr=err.data_ptr() if err is not None else 0, stream=stream)
    torch.cuda.synchronize()
    return out


def expected_places(c, counts, totals):
    pos = torch.cat([torch.arange(t - n, t) for n, t in zip(counts, totals)]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts)).cuda()
    return pos, c.table.long()[seq, pos // c.page], pos % c.page


def check_append(c, rows, heads, counts, totals, qkind, rope, style, half, out, before):
    n = sum(counts)
    pos, pg, off = expected_places(c, counts, totals)
    x = rows[:n].double()
    sc = rope[pos] if rope is not None else None
    y, m = rotated64(x[:, :heads + c.kvh], sc, style, half) if rope is not None else (x[:, :heads + c.kvh], x[:, :heads + c.kvh].abs())

    def near(got, want, mag, kind):
        tol = U[kind] * want.abs() + 2.0 ** -22 * mag + (2.0 ** -25 if kind == "f16" else 0)
        assert bool(((got.double() - want).abs() <= tol).all())

    near(out[:n], y[:, :heads], m[:, :heads], qkind)
    assert bool((out[n:] == 9).all())
    v = rows[:n, heads + c.kvh:]
    if c.kind == "q8_0":
        y32 = rotated32(rows[:n, heads:heads + c.kvh], sc, style, half) if rope is not None else rows[:n, heads:heads + c.kvh].float().cpu().numpy()
        for val, scl, ref in ((c.k, c.ks, y32), (c.v, c.vs, v.float().cpu().numpy())):
            q, bits = quantised(ref)
            assert np.array_equal(val[pg, :, off].cpu().numpy(), q)
            assert np.array_equal(scl[pg, :, off].contiguous().view(torch.int16).cpu().numpy().view(np.uint16), bits)
    else:
        near(c.k[pg, :, off], y[:, heads:], m[:, heads:], c.kind)
        near(c.v[pg, :, off], v.double(), v.double().abs(), c.kind)
    # every other place is as it was
    for now, was in zip((c.k, c.v, c.ks, c.vs), before):
        if now is None:
            continue
        mask = torch.ones(now.shape[:3], dtype=torch.bool, device="cuda")
        mask[pg, :, off] = False
        bits = {1: torch.int8, 2: torch.int16}[now.element_size()]
        assert torch.equal(now.contiguous().view(bits)[mask], was.contiguous().view(bits)[mask])


@pytest.mark.parametrize("kind", ["f16", "bf16", "q8_0"])
@pytest.mark.parametrize("inkind,qkind", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("heads,kvh,hd,page,style,half", [(4, 2, 64, 16, "pairs", 32), (3, 1, 128, 8, "halves", 64), (8, 2, 64, 64, "halves", 32),
                                                          (6, 3, 128, 32, "pairs", 64), (64, 8, 128, 16, "pairs", 22), (0, 2, 64, 8, "pairs", 10)])
def test_append(ncm, cuda, kind, inkind, qkind, heads, kvh, hd, page, style, half):
    counts, totals = [1, 0, 5, 33, 2], [1, 7, 40, 33, 300]
    c = Cache(ncm, kind, kvh, hd, page, totals, seed=heads * 3 + hd)
    before = [x.clone() if x is not None else None for x in (c.k, c.v, c.ks, c.vs)]
    rows = (torch.randn((sum(counts) + 3, heads + 2 * kvh, hd), generator=c.g, device="cuda") * 3).to(DT[inkind])
    rows[2, :, :32] = 0.0   # a block of zeros has scale 0
    rope = rope_table(max(totals), half, hd)
    out = append(ncm, c, rows, heads, counts, totals, qkind, inkind, rope, style, half)
    check_append(c, rows, heads, counts, totals, qkind, rope, style, half, out, before)


@pytest.mark.parametrize("batch", [1, 31, 32, 33, 1023, 1100])
def test_append_one_token_each_and_packed_agree(ncm, cuda, batch):
    """One row per sequence with and without cu_tokens; the search over cu_tokens at its borders."""
    totals = [1 + (7 * i) % 50 for i in range(batch)]
    c = Cache(ncm, "bf16", 1, 64, 8, totals, seed=batch)
    before = [c.k.clone(), c.v.clone(), None, None]
    rows = torch.randn((batch, 4, 64), generator=c.g, device="cuda").bfloat16()
    rope = rope_table(60, 32, 64)
    out = append(ncm, c, rows, 2, [1] * batch, totals, "bf16", "bf16", rope, "pairs", 32, cu=False)
    check_append(c, rows, 2, [1] * batch, totals, "bf16", rope, "pairs", 32, out, before)
    k, v = c.k.clone(), c.v.clone()
    again = append(ncm, c, rows, 2, [1] * batch, totals, "bf16", "bf16", rope, "pairs", 32)
    assert torch.equal(out, again) and torch.equal(k.nan_to_num(5.0), c.k.nan_to_num(5.0)) and torch.equal(v.nan_to_num(5.0), c.v.nan_to_num(5.0))


def test_append_without_rotation_in_place_and_interleaved(ncm, cuda):
    counts, totals = [9, 4], [9, 20]
    c = Cache(ncm, "f16", 2, 64, 16, totals, seed=1, interleaved=True)
    before = [c.k.clone(), c.v.clone(), None, None]
    rows = torch.randn((13, 8, 64), generator=c.g, device="cuda").half()
    out = append(ncm, c, rows, 4, counts, totals, "f16", "f16", None, "pairs", 0)
    check_append(c, rows, 4, counts, totals, "f16", None, "pairs", 0, out, before)
    q, k = torch.randn((13, 4, 64), generator=c.g, device="cuda").half(), torch.randn((13, 2, 64), generator=c.g, device="cuda").half()
    rope, x = rope_table(20, 32, 64), q.clone()
    keep = int32([0, 9, 13]), int32(totals)
    ncm.paged_append(c.kv, ncm.F16, q.data_ptr(), k.data_ptr(), k.data_ptr(), q.data_ptr(), ncm.F16, 13, 4, 2,
                     keep[0].data_ptr(), keep[1].data_ptr(), c.table.data_ptr(), c.width, rope.data_ptr(), 20, 32)
    y, m = rotated64(x.double(), rope[expected_places(c, counts, totals)[0]], "pairs", 32)
    assert bool(((q.double() - y).abs() <= U["f16"] * y.abs() + 2.0 ** -22 * m + 2.0 ** -25).all())


def test_append_out_of_range_rows_are_not_written(ncm, cuda):
    """A position before 0, past the page table or past the rotation table, a bad page id."""
    heads, kvh, hd = 2, 1, 64
    rope = rope_table(30, 32, 64)
    for counts, totals, page_at in (([5, 3], [3, 10], None), ([5, 3], [5, 49], None), ([5, 3], [5, 32], None), ([5, 3], [5, 10], -1), ([5, 3], [5, 10], 1 << 20)):
        c = Cache(ncm, "bf16", kvh, hd, 8, [16, 48], seed=3)
        if page_at is not None:
            c.table[1, 1] = page_at   # positions 8 to 15
        rows, err = torch.randn((8, 4, hd), generator=c.g, device="cuda").bfloat16(), int32([0])
        out = append(ncm, c, rows, heads, counts, totals, "bf16", "bf16", rope, "pairs", 32, err=err)
        assert err.item() == ncm.DEVICE_BAD_ARG
        pos = [t - n + i for n, t in zip(counts, totals) for i in range(n)]
        seq = [0] * 5 + [1] * 3
        good = [0 <= p < min(30, 8 * c.width) and not (page_at is not None and s == 1 and 8 <= p < 16) for p, s in zip(pos, seq)]
        assert [bool((out[i] != 9).any()) for i in range(8)] == good
        assert int((~c.k.isnan()).sum()) == sum(good) * kvh * hd


def test_append_then_attend(ncm, cuda):
    """A batch as it is served: prompts appended, then steps of append and attention, captured."""
    heads, kvh, hd, page, prompts, steps = 8, 2, 128, 16, [37, 1, 200], 5
    c = Cache(ncm, "bf16", kvh, hd, page, [n + steps for n in prompts], seed=21)
    rope = rope_table(256, 64, 128)
    rows = torch.randn((sum(prompts), heads + 2 * kvh, hd), generator=c.g, device="cuda").bfloat16()
    append(ncm, c, rows, heads, prompts, prompts, "bf16", "bf16", rope, "pairs", 64)
    lengths, step = int32(prompts), torch.zeros((3, heads + 2 * kvh, hd), device="cuda").bfloat16()
    q, out = (torch.zeros((3, heads, hd), device="cuda").bfloat16() for _ in range(2))
    space = torch.zeros(ncm.paged_attention_workspace(heads, kvh, hd), dtype=torch.uint8, device="cuda")
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        es, w = 2, (heads + 2 * kvh) * hd
        ncm.paged_append(c.kv, ncm.BF16, step.data_ptr(), step.data_ptr() + es * heads * hd, step.data_ptr() + es * (heads + kvh) * hd,
                         q.data_ptr(), ncm.BF16, 3, heads, 3, 0, lengths.data_ptr(), c.table.data_ptr(), c.width, rope.data_ptr(),
                         256, 64, q_stride=w, k_stride=w, v_stride=w, stream=s.cuda_stream)
        attend(ncm, c, q, lengths, heads, "bf16", out=out, space=space, stream=s.cuda_stream)
    for i in range(steps):
        lengths += 1
        step.copy_(torch.randn(step.shape, generator=c.g, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        n = [p + i + 1 for p in prompts]
        pos = torch.tensor(n).cuda() - 1
        y, m = rotated64(step[:, :heads].double(), rope[pos], "pairs", 64)
        assert bool(((q.double() - y).abs() <= U["bf16"] * y.abs() + 2.0 ** -22 * m).all())
        check(c, q, out, n, "bf16")
