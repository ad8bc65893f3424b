"""The batched serving operators at the ends of their ranges, against plain forms in 64 bits.

Tolerances are those of test_gpu_paged and test_gpu_prompt but for the terms that the tests state.
Over Q8_0 include/ncm.h has each weight, p times scale, as a multiple of at most 1/65000 of the
largest such product among 32 keys (from a multiple of 32 on): it is off by 1/130000 of that, times a
value of at most 127, for each of the 32."""
import pytest
import torch

from test_gpu_paged import DT, U, Cache, append, attend, attend64 as attend_one, check as check_one, check_append, int32, rope_table
from test_gpu_prompt import E, attend as attend_prompt, attend64 as attend_all, check as check_prompt, inputs, starts

pytestmark = pytest.mark.gpu


def attend_q8(q, k, v, v_scales, scale, qkind):
    """attend_one over a Q8_0 cache, with the term of the weights by their products."""
    heads, hd = q.shape
    g = heads // k.shape[1]
    o, _ = attend_one(q, k, v, scale, qkind, hd)
    kr, vr = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    w = torch.softmax(torch.einsum("hd,nhd->hn", q.double(), kr) * scale, -1)
    a = torch.einsum("hn,nhd->hd", w, vr.abs())
    top = (torch.einsum("hd,nhd->hn", q.double().abs(), kr.abs()) * scale).amax(-1)[:, None]
    step = q.double().abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1) / 65024
    e = 2 * (2.0 ** -24 * (hd + 4) * top + 2.0 ** -21) + k.shape[0] * 2.0 ** -24
    e = e + 2 * (torch.einsum("hd,nhd->hn", step, kr.abs()) * scale).amax(-1)[:, None]
    prod = w.T[:, :, None] * v_scales.double().repeat_interleave(g, 1)                                      # [n, heads, hd / 32]
    prod = torch.nn.functional.pad(prod, (0, 0, 0, 0, 0, -k.shape[0] % 32)).unflatten(0, (-1, 32)).amax(1)  # [units, heads, hd / 32]
    return o, U[qkind] * o.abs() + e * a * (1 + U[qkind]) + prod.sum(0).repeat_interleave(32, -1) * (32 * 127 / 130000)


@pytest.mark.parametrize("qkind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 64), (8, 2, 128), (12, 1, 64), (24, 2, 128)])
@pytest.mark.parametrize("lengths", [[32, 77, 3000], [1000] * 40, [20000]])
@pytest.mark.parametrize("less", [1, 100, 1000])
def test_q8_weights_of_a_sink(ncm, cuda, qkind, heads, kvh, hd, lengths, less):
    """One key takes nearly all weight and its value is small, as the first token of a text does."""
    c = Cache(ncm, "q8_0", kvh, hd, 16, lengths, seed=hd + less).fill()
    q = (torch.rand((len(lengths), heads, hd), generator=c.g, device="cuda") + 0.5).to(DT[qkind])
    for i, n in enumerate(lengths):
        at = 5 if i % 2 else n - 1 - n // 3
        page, off = c.table[i, at // 16].item(), at % 16
        c.k[page, :, off] = 100
        c.ks[page, :, off] = 0.011 if hd == 128 else 0.016    # a score of about 12 over the others': 2^-18 and up of its weight
        c.vs[page, :, off] = torch.as_tensor(0.01 / less).half()
    out = attend(ncm, c, q, int32(lengths), heads, qkind)
    for i, n in enumerate(lengths):
        ref, tol = attend_q8(q[i], c.rows("k", i, n), c.rows("v", i, n), c.rows("v_scales", i, n), hd ** -0.5, qkind)
        off = (out[i].double() - ref).abs()
        assert bool((off <= tol).all()), (i, n, float((off / tol).max()), float((off / ref.abs().mean()).max()))


@pytest.mark.parametrize("n", [5, 40, 3000, 40000])
@pytest.mark.parametrize("hd", [64, 128])
def test_q8_not_finite(ncm, cuda, n, hd):
    """Scores that are all -infinity give zeros; a NaN in a key's or a value's scale or in a query
    reaches its outputs and no others."""
    heads, kvh = 8, 2
    c = Cache(ncm, "q8_0", kvh, hd, 64, [n, 50], seed=13).fill()
    pages, lengths = c.table[0, :-(-n // 64)].long(), int32([n, 50])
    q = torch.rand((2, heads, hd), generator=c.g, device="cuda").bfloat16() + 1
    good = attend(ncm, c, q, lengths, heads, "bf16")
    assert bool(good.isfinite().all())
    page, off = c.table[0, (n - 1) // 2 // 64].item(), (n - 1) // 2 % 64
    for plane in (c.ks, c.vs):
        keep = plane[page, 1, off, 1].clone()
        plane[page, 1, off, 1] = float("nan")
        out = attend(ncm, c, q, lengths, heads, "bf16")
        plane[page, 1, off, 1] = keep
        assert torch.equal(out[1], good[1]) and torch.equal(out[0, :4], good[0, :4])
        block = out[0, 4:] if plane is c.ks else out[0, 4:, 32:64]
        assert bool(block.isnan().all())
        if plane is c.vs:
            assert torch.equal(out[0, 4:, :32], good[0, 4:, :32]) and torch.equal(out[0, 4:, 64:], good[0, 4:, 64:])
    bad = q.clone()
    bad[0, 2, 7] = float("nan")
    out = attend(ncm, c, bad, lengths, heads, "bf16")
    rest = [0, 1, 3, 4, 5, 6, 7]
    assert bool(out[0, 2].isnan().all()) and torch.equal(out[0, rest], good[0, rest]) and torch.equal(out[1], good[1])
    c.k[pages] = -1
    c.ks[pages] = float("inf")
    out = attend(ncm, c, q, lengths, heads, "bf16")
    assert bool((out[0] == 0).all()) and torch.equal(out[1], good[1])


@pytest.mark.parametrize("less", [12.5, 4.5, 1.5, 0.45])
def test_f16_many_small_weights(ncm, cuda, less):
    """A key of weight one and 2^18 of `less` x 2^-24 each: together they matter, and each lies among
    f16's subnormal numbers or below them.  Held times 2^7, one below 2^-21 is off by 2^-32, half a
    step of those numbers."""
    n, hd, heads = 1 << 18, 64, 8
    k, v = torch.zeros((n, hd), device="cuda").half(), torch.ones((n, hd), device="cuda").half()
    at = 12345
    q = torch.ones((1, heads, hd), device="cuda").half()
    # scale * q.k = ln 2 * (24 - log2 less), to f16's precision; the sink's value is zero
    k[at], v[at] = (24 - torch.log2(torch.tensor(less)).item()) * 0.6931471805599453 / 8.0, 0.0
    c = Cache(ncm, "f16", 1, hd, 64, [n], seed=1)
    order = c.table[0].long()
    c.k[order, 0], c.v[order, 0] = k.view(-1, 64, hd), v.view(-1, 64, hd)
    s = q[0, 0].double() @ k.double().T * 0.125
    w = torch.softmax(s, -1)
    o = (w @ v.double())[0].item()
    e = 2 * (2.0 ** -24 * (hd + 4) * s.abs().max().item() + 2.0 ** -21) + n * 2.0 ** -24 + E["f16"]
    tol = U["f16"] * o + (U["f16"] + e) * o * (1 + U["f16"]) + n * 2.0 ** -32
    out = attend(ncm, c, q, int32([n]), heads, "f16")
    assert bool(((out.double() - o).abs() <= tol).all()), (float(out[0, 0, 0]), o, tol)
    out = attend_prompt(ncm, q, k[:, None], v[:, None], int32([0, 1]), int32([0, n]), "f16", True)
    assert bool(((out.double() - o).abs() <= tol).all()), (float(out[0, 0, 0]), o, tol)


@pytest.mark.parametrize("n", [5, 40, 3000, 40000])
def test_all_scores_minus_infinity_over_values_that_are_not_finite(ncm, cuda, n):
    """Zeros, whatever the values hold: whole segments, parts joined in a CTA and over few and many."""
    heads, kvh, hd = 8, 2, 64
    for kind in ("bf16", "f16"):
        c = Cache(ncm, kind, kvh, hd, 64, [n, 50], seed=13).fill()
        q = torch.rand((2, heads, hd), generator=c.g, device="cuda").to(DT[kind]) + 1
        good = attend(ncm, c, q, int32([n, 50]), heads, kind)
        pages = c.table[0, :-(-n // 64)].long()
        c.k[pages], c.v[pages] = float("-inf"), float("inf")
        c.v[pages, :, 3] = float("nan")
        out = attend(ncm, c, q, int32([n, 50]), heads, kind)
        assert bool((out[0] == 0).all()) and torch.equal(out[1], good[1])


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_prompt_all_scores_minus_infinity_over_values_that_are_not_finite(ncm, cuda, kind):
    lens = [60, 150, 400, 40]
    q, k, v = inputs(lens, lens, 4, 2, 64, kind, seed=9)
    q, cu = q.abs() + 1, int32(starts(lens))
    good = attend_prompt(ncm, q, k, v, cu, cu, kind, True)
    k[60:610], v[60:610] = float("-inf"), float("inf")
    v[60:610:7] = float("nan")
    for causal in (True, False):
        out = attend_prompt(ncm, q, k, v, cu, cu, kind, causal)
        assert bool((out[60:610] == 0).all())
        if causal:
            assert torch.equal(out[:60], good[:60]) and torch.equal(out[610:], good[610:])


def cut(cu, total):
    """Starts raised to the largest before them and cut to the range."""
    out = []
    for x in cu:
        out.append(min(max([x, 0] + out), total))
    return out


@pytest.mark.parametrize("heads,kvh,hd", [(4, 1, 128), (8, 2, 64)])
@pytest.mark.parametrize("cu", [[0, 2000, 0, 2000], [0, 1000, 20, 1500, 1400], [0, 1700, 5, 1800, 6, 1900, 7, 1950], [300, 200, 900, 2 ** 31 - 1, 0, 2000],
                                [-5, 700, -2 ** 31, 1200]])
def test_prompt_falling_starts(ncm, cuda, heads, kvh, hd, cu):
    """A sequence whose start falls below an earlier one's end begins there: rows have one sequence
    each, the sound ones are right, and rows of none are left alone."""
    total, err = 2000, int32([0])
    q, k, v = inputs([total], [total], heads, kvh, hd, "bf16", seed=len(cu))
    clean = cut(cu, total)
    lk = [200 + 7 * i for i in range(len(cu) - 1)]
    k, v = k[:sum(lk)], v[:sum(lk)]
    lq, a = [y - x for x, y in zip(clean, clean[1:])], clean[0]
    for causal in (False, True):
        err.zero_()
        out = attend_prompt(ncm, q, k, v, int32(cu), int32(starts(lk)), "bf16", causal, err=err)
        assert err.item() == ncm.DEVICE_BAD_ARG
        assert bool((out[:a] == 7).all()) and bool((out[clean[-1]:] == 7).all())
        check_prompt(q[a:], k, v, out[a:], lq, lk, "bf16", causal)


def test_prompt_falling_starts_of_many_sequences(ncm, cuda):
    """The same where the sequences take several launches."""
    batch, total, err = 2500, 5000, int32([0])
    cu = [2 * i for i in range(batch + 1)]
    cu[700], cu[1024], cu[1500], cu[1501] = 4000, 3, 100, 0
    q, k, v = inputs([total], [total], 4, 2, 64, "f16", seed=3)
    clean = cut(cu, total)
    lk = [1 + i % 3 for i in range(batch)]
    lk[-1] += total - sum(lk) if sum(lk) < total else 0
    ck = starts(lk)
    out = attend_prompt(ncm, q, k, v, int32(cu), int32(ck), "f16", False, err=err)
    assert err.item() == ncm.DEVICE_BAD_ARG
    for i in list(range(0, batch, 83)) + [698, 699, 700, 1023, 1024, 1025, 1499, 1500, 1501, 1999, 2000, 2001, 2047, 2048, 2049, 2499]:
        a, b = clean[i], clean[i + 1]
        ref, tol = attend_all(q[a:b], k[ck[i]:ck[i + 1]], v[ck[i]:ck[i + 1]], 0.125, None, "f16")
        assert bool(((out[a:b].double() - ref).abs() <= tol).all()), i


@pytest.mark.parametrize("cu", [[0, 5, 3, 2, 8], [0, 9, 1, 2, 8], [0, -3, 2, 2, 8], [0, 2, 4, 6, 9], [2 ** 31 - 1, -2 ** 31, 0, 0, 8],
                                [0, 2, 4, 2 ** 31 - 1, 8], [-1, 2, 4, 6, 8]])
def test_append_bad_starts_are_flagged(ncm, cuda, cu):
    """Starts that fall or lie out of range: flagged, and a row is stored only where the sequence that
    the definition gives it to (cu[s] <= i < cu[s + 1]) has its place."""
    batch, tokens, heads, kvh, hd, page = 4, 8, 2, 1, 64, 8
    totals = [20, 25, 30, 35]
    c = Cache(ncm, "bf16", kvh, hd, page, [48] * batch, seed=3)
    rows, err = torch.randn((tokens, heads + 2 * kvh, hd), generator=c.g, device="cuda").bfloat16(), int32([0])
    keep, out = (int32(cu), int32(totals)), torch.full((tokens, heads, hd), 9.0, device="cuda").bfloat16()
    w, es = (heads + 2 * kvh) * hd, 2
    ncm.paged_append(c.kv, ncm.BF16, rows.data_ptr(), rows.data_ptr() + es * heads * hd, rows.data_ptr() + es * (heads + kvh) * hd, out.data_ptr(),
                     ncm.BF16, tokens, heads, batch, keep[0].data_ptr(), keep[1].data_ptr(), c.table.data_ptr(), c.width, q_stride=w, k_stride=w,
                     v_stride=w, err_ptr=err.data_ptr())
    torch.cuda.synchronize()
    assert err.item() == ncm.DEVICE_BAD_ARG
    allowed = torch.zeros((c.pages, page), dtype=torch.bool, device="cuda")
    for s in range(batch):
        for i in range(tokens):
            if cu[s] <= i < cu[s + 1]:
                pos = totals[s] - cu[s + 1] + i
                if 0 <= pos < 48:
                    allowed[c.table[s, pos // page].item(), pos % page] = True
    written = ~c.k[:, 0, :, 0].isnan()
    assert not bool((written & ~allowed).any())


@pytest.mark.parametrize("batch", [3, 33, 700, 1500])
def test_append_falling_start_anywhere_is_flagged(ncm, cuda, batch):
    tokens = 2 * batch
    c = Cache(ncm, "f16", 1, 64, 8, [8] * batch, seed=batch)
    rows, err = torch.randn((tokens, 3, 64), generator=c.g, device="cuda").half(), int32([0])
    cu, lengths, out = int32([2 * i for i in range(batch + 1)]), int32([8] * batch), torch.zeros((tokens, 1, 64), device="cuda").half()

    def call():
        err.zero_()
        ncm.paged_append(c.kv, ncm.F16, rows.data_ptr(), rows.data_ptr() + 128, rows.data_ptr() + 256, out.data_ptr(), ncm.F16, tokens, 1, batch,
                         cu.data_ptr(), lengths.data_ptr(), c.table.data_ptr(), 1, q_stride=192, k_stride=192, v_stride=192, err_ptr=err.data_ptr())
        return err.item()

    assert call() == 0
    for at in {1, batch // 2, batch - 1}:
        keep = cu[at].item()
        cu[at] = keep + 3
        assert call() == ncm.DEVICE_BAD_ARG
        cu[at] = keep
    cu[batch] += 1
    assert call() == ncm.DEVICE_BAD_ARG
    cu[batch] -= 1
    assert call() == 0


def test_prompt_rows_of_no_token_cost_nothing(ncm, cuda):
    """A group of 12 fills 120 of a tile's 128 rows; the others hold what an earlier kernel left in
    shared memory.  NaN there changes no output, and no time: the sums were rescaled at every step
    for them, which took 1.7 times as long (1.02 without; the best of 20 each)."""
    def call(heads, n, fill):
        q, k, v = inputs([n], [n], heads, 8, 128, "bf16", seed=1)
        if fill is not None:
            q.fill_(fill)
        cu, out = int32([0, n]), torch.empty_like(q)
        return lambda: attend_prompt(ncm, q, k, v, cu, cu, "bf16", True, out=out, stream=torch.cuda.current_stream().cuda_stream)

    f, before, best, outs = call(96, 4000, None), [call(32, 6000, x) for x in (0.0, float("nan"))], [1e9, 1e9], [None, None]
    f()
    for _ in range(20):
        for i in range(2):
            before[i]()
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            out = f()
            b.record()
            outs[i] = out.clone()
            torch.cuda.synchronize()
            best[i] = min(best[i], a.elapsed_time(b))
    assert torch.equal(*outs)
    assert best[1] < 1.3 * best[0], best


def test_host_pointers_are_told_from_sound_ones(ncm, cuda):
    """Calls that succeed, and then each of their pointers in turn in host memory, refused for that."""
    host = torch.zeros(1 << 16, dtype=torch.uint8).pin_memory().data_ptr()
    space = torch.zeros(ncm.paged_attention_workspace(2, 1, 64), dtype=torch.uint8, device="cuda")
    x = [torch.ones(16 * 64 * 4, dtype=torch.float16, device="cuda") for _ in range(8)]
    q, k, v, out, pk, pv, sk, sv = (t.data_ptr() for t in x)
    starts_, lengths, table, err = int32([0, 1]), int32([1]), int32([0]), int32([0])
    rope = torch.ones((1, 32, 2), device="cuda")

    def each(f, base, names):
        f(**base)
        torch.cuda.synchronize()
        assert err.item() == 0
        for name in names or [n for n in base if n.endswith("_ptr")]:
            with pytest.raises(ncm.NcmError, match="not a device pointer"):
                f(**{**base, name: host})

    kv = ncm.PagedKV(ncm.F16, pk, pv, 4, 16, 1, 64)
    each(lambda **a: ncm.paged_append(kv, **a),
         dict(in_type=ncm.F16, q_ptr=q, k_ptr=k, v_ptr=v, q_out_ptr=out, q_out_type=ncm.F16, tokens=1, heads=2, batch=1, cu_tokens_ptr=starts_.data_ptr(),
              lengths_ptr=lengths.data_ptr(), page_table_ptr=table.data_ptr(), table_width=1, rope_ptr=rope.data_ptr(), rope_len=1, rope_half=32,
              err_ptr=err.data_ptr()), None)
    decode = dict(q_type=ncm.F16, batch=1, heads=2, lengths_ptr=lengths.data_ptr(), page_table_ptr=table.data_ptr(), table_width=1,
                  workspace_ptr=space.data_ptr(), workspace_bytes=space.numel(), err_ptr=err.data_ptr())
    each(lambda out_ptr=out, q_ptr=q, **a: ncm.paged_attention(out_ptr, q_ptr, kv, **a), {**decode, "out_ptr": out, "q_ptr": q}, None)

    def over(k=pk, v=pv, k_scales=sk, v_scales=sv, **a):
        ncm.paged_attention(out, q, ncm.PagedKV(ncm.Q8_0, k, v, 4, 16, 1, 64, k_scales, v_scales), **a)

    each(over, decode, ["k", "v", "k_scales", "v_scales"])
    each(lambda **a: ncm.prompt_attention(**a),
         dict(out_ptr=out, q_ptr=q, k_ptr=k, v_ptr=v, type=ncm.F16, total_q=1, total_k=1, batch=1, heads=2, kv_heads=1, head_dim=64,
              cu_q_ptr=starts_.data_ptr(), cu_k_ptr=starts_.data_ptr(), err_ptr=err.data_ptr()), None)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kvh,hd", [(65, 1, 64), (100, 1, 128), (127, 1, 128), (128, 1, 64), (256, 2, 128), (43, 1, 64)])
def test_prompt_wide_groups(ncm, cuda, kind, heads, kvh, hd):
    """One to a few tokens to a tile."""
    lq, lk = [5, 0, 1, 40], [5, 3, 200, 333]
    q, k, v = inputs(lq, lk, heads, kvh, hd, kind, seed=heads, rows_behind=2)
    for causal in (True, False):
        out = attend_prompt(ncm, q, k, v, int32(starts(lq)), int32(starts(lk)), kind, causal)
        check_prompt(q, k, v, out, lq, lk, kind, causal)
        assert bool((out[sum(lq):] == 7).all())


@pytest.mark.parametrize("kind,qkind", [("bf16", "bf16"), ("q8_0", "f16")])
@pytest.mark.parametrize("heads,kvh,hd", [(17, 1, 64), (33, 1, 128), (128, 1, 128), (100, 2, 64), (600, 600, 64)])
def test_attention_wide_groups(ncm, cuda, kind, qkind, heads, kvh, hd):
    """Groups that make several segments, and many key-value heads."""
    lengths = [0, 1, 33, 700] if kvh < 600 else [3, 40]
    c = Cache(ncm, kind, kvh, hd, 16, lengths, seed=heads).fill()
    q = torch.randn((len(lengths), heads, hd), generator=c.g, device="cuda").to(DT[qkind])
    check_one(c, q, attend(ncm, c, q, int32(lengths), heads, qkind), lengths, qkind)


@pytest.mark.parametrize("hd", [64, 128])
def test_q8_outlier_channel_in_q(ncm, cuda, hd):
    """One value of a block of q many times the others, which its integers are multiples of."""
    lengths, heads, kvh = [40, 2000], 8, 2
    c = Cache(ncm, "q8_0", kvh, hd, 32, lengths, seed=4).fill()
    for times in (20, 1000):
        q = torch.randn((2, heads, hd), generator=c.g, device="cuda")
        q[:, :, 37] *= times
        q = q.half()
        check_one(c, q, attend(ncm, c, q, int32(lengths), heads, "f16"), lengths, "f16")


@pytest.mark.parametrize("hd", [64, 128])
def test_q8_pages_of_keys_and_values_side_by_side(ncm, cuda, hd):
    """A Q8_0 cache in one allocation with a page stride: append, then attention."""
    heads, kvh, page, totals = 8, 2, 16, [50, 3, 130]
    c = Cache(ncm, "q8_0", kvh, hd, page, totals, seed=2)
    both = torch.full((c.pages, 2, kvh, page, hd), 127, dtype=torch.int8, device="cuda")
    c.k, c.v = both[:, 0], both[:, 1]
    c.kv = ncm.PagedKV(ncm.Q8_0, c.k.data_ptr(), c.v.data_ptr(), c.pages, page, kvh, hd, c.ks.data_ptr(), c.vs.data_ptr(), 2 * kvh * page * hd)
    before = [x.clone() for x in (c.k, c.v, c.ks, c.vs)]
    rows = torch.randn((sum(totals), heads + 2 * kvh, hd), generator=c.g, device="cuda").half()
    rope = rope_table(200, hd // 2, hd)
    out = append(ncm, c, rows, heads, totals, totals, "f16", "f16", rope, "halves", hd // 2)
    check_append(c, rows, heads, totals, totals, "f16", rope, "halves", hd // 2, out, before)
    q = out[[49, 52, 182]].contiguous()
    check_one(c, q, attend(ncm, c, q, int32(totals), heads, "f16"), totals, "f16")


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("inkind", ["f32", "bf16"])
def test_append_many_tokens_in_several_passes(ncm, cuda, kind, inkind):
    """So many tokens that a CTA takes each in passes of 128 threads."""
    counts, totals, heads, kvh, hd = [700, 1, 0, 333], [700, 50, 9, 400], 24, 6, 128
    c = Cache(ncm, kind, kvh, hd, 32, totals, seed=6)
    before = [x.clone() if x is not None else None for x in (c.k, c.v, c.ks, c.vs)]
    rows = (torch.randn((sum(counts) + 5, heads + 2 * kvh, hd), generator=c.g, device="cuda") * 2).to(DT[inkind])
    rope = rope_table(700, 64, hd)
    out = append(ncm, c, rows, heads, counts, totals, "bf16", inkind, rope, "pairs", 64)
    check_append(c, rows, heads, counts, totals, "bf16", rope, "pairs", 64, out, before)


def test_rows_and_pages_past_32_bits(ncm, cuda):
    """Elements past 2^31 and bytes past 2^32 of each operator's rows, and of the append's pages."""
    heads, kvh, hd, n, apart = 4, 2, 64, 100, 1 << 25
    wide = torch.zeros(n * apart, dtype=torch.float16, device="cuda").view(n, apart)
    g = torch.Generator(device="cuda").manual_seed(3)
    wide[:, :2 * heads * hd + 2 * kvh * hd] = torch.randn((n, 2 * heads * hd + 2 * kvh * hd), generator=g, device="cuda").half()
    at = [0, heads * hd, (heads + kvh) * hd, (heads + 2 * kvh) * hd]
    q, k, v, out = (wide[:, a:a + h * hd].unflatten(1, (h, hd)) for a, h in zip(at, (heads, kvh, kvh, heads)))
    cu = int32([0, 30, n])
    ncm.prompt_attention(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), ncm.F16, n, n, 2, heads, kvh, hd, cu.data_ptr(), cu.data_ptr(),
                         q_stride=apart, k_stride=apart, v_stride=apart, out_stride=apart)
    check_prompt(q, k, v, out, [30, 70], [30, 70], "f16", True)
    page = 8
    pages = 2 ** 31 // (kvh * page * hd) + 20
    c = Cache(ncm, "f16", kvh, hd, page, [60, 60], seed=1)
    c.k, c.v = (torch.full((pages, kvh, page, hd), 3.0, dtype=torch.float16, device="cuda") for _ in range(2))
    c.pages, c.kv = pages, ncm.PagedKV(ncm.F16, c.k.data_ptr(), c.v.data_ptr(), pages, page, kvh, hd)
    c.table = torch.randperm(16, generator=g, device="cuda").to(torch.int32).view(2, 8).contiguous()
    c.table[:, 4:] += pages - 16
    cu, lengths, q_out, err = int32([0, 40, n]), int32([40, 60]), torch.zeros((n, heads, hd), dtype=torch.float16, device="cuda"), int32([0])
    ncm.paged_append(c.kv, ncm.F16, q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), ncm.F16, n, heads, 2, cu.data_ptr(), lengths.data_ptr(),
                     c.table.data_ptr(), 8, q_stride=apart, k_stride=apart, v_stride=apart, err_ptr=err.data_ptr())
    assert err.item() == 0 and torch.equal(q_out, q)
    assert torch.equal(c.rows("k", 0, 40), k[:40].double()) and torch.equal(c.rows("v", 1, 60), v[40:].double())
    space = torch.zeros(ncm.paged_attention_workspace(heads, kvh, hd), dtype=torch.uint8, device="cuda")
    ncm.paged_attention(out[39].data_ptr(), q[39].data_ptr(), c.kv, ncm.F16, 2, heads, lengths.data_ptr(), c.table.data_ptr(), 8, space.data_ptr(),
                        space.numel(), q_stride=60 * apart, out_stride=60 * apart)
    for i, row in enumerate((39, 99)):
        ref, tol = attend_one(q[row], c.rows("k", i, (40, 60)[i]), c.rows("v", i, (40, 60)[i]), hd ** -0.5, "f16", hd)
        assert bool(((out[row].double() - ref).abs() <= tol).all())


def test_scores_that_overflow_are_not_zeros(ncm, cuda):
    """A score past f32's range, by the scale or by itself, makes its row NaN in both operators."""
    heads, kvh, hd = 4, 2, 64
    for n in (7, 3000):
        c = Cache(ncm, "bf16", kvh, hd, 16, [n, 40], seed=2).fill()
        q = torch.randn((2, heads, hd), generator=c.g, device="cuda").bfloat16()
        good = attend(ncm, c, q, int32([n, 40]), heads, "bf16", scale=30.0)
        at = n // 2
        page, off = c.table[0, at // 16].item(), at % 16
        c.k[page, 1, off] = 2e18
        q[0, 2:] = 1e18   # q.k = 1.3e38, times 30 past the range
        for scale in (30.0, 1e10):
            out = attend(ncm, c, q, int32([n, 40]), heads, "bf16", scale=scale)
            assert bool(out[0, 2:].isnan().all())
            assert scale != 30.0 or torch.equal(out[0, :2], good[0, :2]) and torch.equal(out[1], good[1])
        k, v = c.rows("k", 0, n).bfloat16(), c.rows("v", 0, n).bfloat16()
        out = attend_prompt(ncm, q[:1], k, v, int32([0, 1]), int32([0, n]), "bf16", True, scale=30.0)
        assert bool(out[0, 2:].isnan().all())
