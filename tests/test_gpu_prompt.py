"""Attention over whole packed prompts against the plain form in 64 bits.

Tolerances as for one token (test_gpu_paged): with u half a step of the output's type, an output
o = sum w_j v_j carries u |o| for its own rounding, u sum w_j |v_j| for the roundings of p, the
f32 error of the scores, e = 2 (2^-24 (head_dim + 4) max |q||k| scale + 2^-21) relative to each
w_j, n 2^-24 for the sums, and for f16 the 2^-25 that a p below 2^-14 may be off.  An exponential
computed by a polynomial is off by at most 2^-13.7 (bf16) or 2^-18.4 (f16), relative, which
counts twice, in p and in its sum."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
E = {"bf16": 2.0 ** -12.7, "f16": 2.0 ** -17.4}
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def attend64(q, k, v, scale, shift, kind):
    """q [n, H, d] over k, v [m, KH, d] in 64 bits; row i sees keys up to i + shift (None: all)."""
    n, heads, d = q.shape
    m, g = k.shape[0], heads // k.shape[1]
    out, tol = (torch.zeros((n, heads, d), dtype=torch.float64, device="cuda") for _ in range(2))
    if m == 0 or n == 0:
        return out, tol
    seen = torch.ones((n, m), dtype=torch.bool, device="cuda") if shift is None else (
        torch.arange(m, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + shift)
    some = seen.any(-1)
    for h in range(heads):
        kh, vh, qh = k[:, h // g].double(), v[:, h // g].double(), q[:, h].double()
        s = (qh @ kh.T) * scale
        s = s.masked_fill(~seen, float("-inf"))
        top = ((qh.abs() @ kh.abs().T) * scale).where(seen, 0.0).amax(-1)[:, None]
        w = torch.softmax(s, -1).where(seen, 0.0)
        o, a = w @ vh, w @ vh.abs()
        u = U[kind]
        e = 2 * (2.0 ** -24 * (d + 4) * top + 2.0 ** -21) + m * 2.0 ** -24 + E[kind]
        small = 2.0 ** -25 * (1 + m * vh.abs().amax()) if kind == "f16" else 0.0
        out[:, h], tol[:, h] = o, u * o.abs() + (u + e) * a * (1 + u) + small
    out[~some], tol[~some] = 0.0, 0.0
    return out, tol


def inputs(lq, lk, heads, kvh, hd, kind, seed, q_scale=1.0, rows_behind=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (torch.randn((sum(lq) + rows_behind, heads, hd), generator=g, device="cuda") * q_scale).to(DT[kind])
    k = torch.randn((sum(lk) + rows_behind, kvh, hd), generator=g, device="cuda").to(DT[kind])
    v = torch.randn((sum(lk) + rows_behind, kvh, hd), generator=g, device="cuda").to(DT[kind])
    return q, k, v


def attend(ncm, q, k, v, cu_q, cu_k, kind, causal, out=None, scale=0.0, err=None, stream=0, **strides):
    out = torch.full_like(q, 7.0) if out is None else out
    ncm.prompt_attention(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), ncm.BF16 if kind == "bf16" else ncm.F16,
                         q.shape[0], k.shape[0], cu_q.numel() - 1, q.shape[1], k.shape[1], q.shape[2], cu_q.data_ptr(),
                         cu_k.data_ptr(), causal=causal, scale=scale, err_ptr=err.data_ptr() if err is not None else 0,
                         stream=stream, **strides)
    return out


def check(q, k, v, out, lq, lk, kind, causal, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    aq, ak = starts(lq), starts(lk)
    for i in range(len(lq)):
        ref, tol = attend64(q[aq[i]:aq[i + 1]], k[ak[i]:ak[i + 1]], v[ak[i]:ak[i + 1]], scale, lk[i] - lq[i] if causal else None, kind)
        off = (out[aq[i]:aq[i + 1]].double() - ref).abs()
        assert bool((off <= tol).all()), (i, lq[i], lk[i], float((off - tol).max()), float(off.max()))


LENGTHS = [([1], [1]), ([128], [128]), ([3, 0, 1, 77, 129], [3, 0, 1, 77, 129]), ([64, 65, 63], [64, 65, 63]), ([1000], [1000]),
           ([5, 130, 0, 257], [133, 130, 9, 300]), ([300, 4, 7], [100, 0, 6]), ([1, 1, 1], [500, 128, 129])]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kvh,hd", [(4, 1, 128), (4, 2, 64), (2, 2, 128), (3, 1, 64), (12, 2, 128), (16, 1, 64), (40, 2, 128)])
@pytest.mark.parametrize("lq,lk", LENGTHS)
def test_prompt_small(ncm, cuda, kind, causal, heads, kvh, hd, lq, lk):
    """One token to a thousand, empty sequences, fewer and more keys than queries, odd groups."""
    q, k, v = inputs(lq, lk, heads, kvh, hd, kind, seed=sum(lq) + heads, rows_behind=2)
    err = int32([0])
    out = attend(ncm, q, k, v, int32(starts(lq)), int32(starts(lk)), kind, causal, err=err)
    check(q, k, v, out, lq, lk, kind, causal)
    assert bool((out[sum(lq):] == 7).all()) and err.item() == 0


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("lq,lk,heads,kvh,hd,causal", [([4000], [4000], 8, 2, 128, True), ([3000], [5000], 8, 1, 64, True),
                                                       ([2048, 1, 999, 3111], [2048, 1, 999, 3111], 8, 2, 64, True),
                                                       ([700, 900], [2300, 6000], 4, 4, 128, False)])
def test_prompt_long(ncm, cuda, kind, lq, lk, heads, kvh, hd, causal):
    """More work than CTAs: each walks over several items, the rings and phases wrap."""
    q, k, v = inputs(lq, lk, heads, kvh, hd, kind, seed=heads, q_scale=2.0)
    cu_q, cu_k = int32(starts(lq)), int32(starts(lk))
    out = attend(ncm, q, k, v, cu_q, cu_k, kind, causal)
    check(q, k, v, out, lq, lk, kind, causal)
    for _ in range(3):
        assert torch.equal(attend(ncm, q, k, v, cu_q, cu_k, kind, causal), out)


def test_prompt_growing_scores(ncm, cuda):
    """Scores that grow along the keys by hundreds, so that the running maximum moves at every tile."""
    n, hd = 1500, 128
    q, k, v = inputs([n], [n], 4, 1, hd, "bf16", seed=2)
    q[:], k[:] = 1.0, torch.linspace(-3, 3, n, device="cuda")[:, None, None].bfloat16()
    q[:, :, 1::4] = -1.0
    for scale in (0.05, 0.7):
        check(q, k, v, attend(ncm, q, k, v, int32([0, n]), int32([0, n]), "bf16", True, scale=scale), [n], [n], "bf16", True, scale)
        check(q, k, v, attend(ncm, q, k, v, int32([0, n]), int32([0, n]), "bf16", False, scale=scale), [n], [n], "bf16", False, scale)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kvh,hd", [(4, 1, 128), (2, 2, 64)])
def test_prompt_hidden_values_do_not_matter(ncm, cuda, kind, heads, kvh, hd):
    """NaN and infinities in keys and values change no row that does not see them, and reach the others."""
    lens = [70, 200, 300]
    q, k, v = inputs(lens, lens, heads, kvh, hd, kind, seed=4, rows_behind=40)
    cu = int32(starts(lens))
    good = attend(ncm, q, k, v, cu, cu, kind, True)
    check(q, k, v, good, lens, lens, kind, True)
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[570:], bad_v[570:] = float("nan"), float("inf")      # behind the last sequence
    assert torch.equal(attend(ncm, q, bad_k, bad_v, cu, cu, kind, True), good)
    for at, key in ((70 + 150, 150), (70 + 30, 30), (70 + 199, 199)):
        bad_v = v.clone()
        bad_v[at, :, 7], bad_v[at, :, hd - 1] = float("inf"), float("nan")
        out = attend(ncm, q, k, bad_v, cu, cu, kind, True)
        assert torch.equal(out[:70], good[:70]) and torch.equal(out[270:], good[270:])
        assert torch.equal(out[70:at], good[70:at])
        mask = torch.ones(hd, dtype=torch.bool, device="cuda")
        mask[7] = mask[hd - 1] = False
        off = (out[at:270][..., mask].double() - good[at:270][..., mask].double()).abs()
        assert bool((off == 0).all())
        assert bool((out[at:270, :, 7] == float("inf")).all()) and bool(out[at:270, :, hd - 1].isnan().all())
        bad_k = k.clone()
        bad_k[at, :, 3] = float("nan")
        out = attend(ncm, q, bad_k, v, cu, cu, kind, True)
        assert torch.equal(out[:at], good[:at]) and torch.equal(out[270:], good[270:]) and bool(out[at:270].isnan().all())


def test_prompt_with_all_scores_minus_infinity(ncm, cuda):
    """Keys of -infinity in the middle sequence: zeros there, the others as they were."""
    lens = [60, 150, 40]
    q, k, v = inputs(lens, lens, 4, 2, 64, "bf16", seed=9)
    q, cu = q.abs() + 1, int32(starts(lens))
    good = attend(ncm, q, k, v, cu, cu, "bf16", True)
    k[60:210] = float("-inf")
    out = attend(ncm, q, k, v, cu, cu, "bf16", True)
    assert bool((out[60:210] == 0).all()) and torch.equal(out[:60], good[:60]) and torch.equal(out[210:], good[210:])


def test_prompt_strides(ncm, cuda):
    """q, k and v as slices of one projection's rows, out rows apart."""
    lens, heads, kvh, hd = [40, 333], 8, 2, 64
    n, wide = sum(lens), heads + 2 * kvh
    rows = torch.randn((n, wide, hd), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
    out = torch.full((n, heads + 1, hd), 7.0, dtype=torch.float16, device="cuda")
    q, k, v = rows[:, :heads], rows[:, heads:heads + kvh], rows[:, heads + kvh:]
    cu = int32(starts(lens))
    attend(ncm, q, k, v, cu, cu, "f16", True, out=out, q_stride=wide * hd, k_stride=wide * hd, v_stride=wide * hd, out_stride=(heads + 1) * hd)
    check(q, k, v, out[:, :heads], lens, lens, "f16", True)
    assert bool((out[:, heads] == 7).all())


def test_prompt_bad_starts_are_cut_and_flagged(ncm, cuda):
    """cu entries that fall or lie out of range touch nothing outside; sound sequences stay right."""
    lens, err = [50, 60, 70], int32([0])
    q, k, v = inputs(lens, lens, 4, 2, 64, "bf16", seed=5)
    good = int32(starts(lens))
    for cu in ([0, 50, 110, 100000], [0, 50, 110, 2 ** 31 - 1], [0, 50, 110, -7], [0, 50, 110, -2 ** 31]):
        for cq, ck in ((int32(cu), good), (good, int32(cu))):
            err.zero_()
            out = attend(ncm, q, k, v, cq, ck, "bf16", True, err=err)
            check(q[:110], k[:110], v[:110], out, lens[:2], lens[:2], "bf16", True)
            assert err.item() == ncm.DEVICE_BAD_ARG


def test_prompt_many_sequences(ncm, cuda):
    """More sequences than one launch takes."""
    lens = [(3 * i) % 5 for i in range(2100)]
    q, k, v = inputs(lens, lens, 4, 2, 64, "f16", seed=6)
    cu = int32(starts(lens))
    out = attend(ncm, q, k, v, cu, cu, "f16", True)
    at = starts(lens)
    for i in list(range(0, 2100, 83)) + [2047, 2048, 2049, 2099]:
        ref, tol = attend64(q[at[i]:at[i + 1]], k[at[i]:at[i + 1]], v[at[i]:at[i + 1]], 0.125, 0, "f16")
        assert bool(((out[at[i]:at[i + 1]].double() - ref).abs() <= tol).all()), i


def test_prompt_without_any_key(ncm, cuda):
    q = torch.randn((5, 4, 64), device="cuda").half()
    out = torch.full_like(q, 7.0)
    cu_q, cu_k = int32([0, 2, 4]), int32([0, 0, 0])
    ncm.prompt_attention(out.data_ptr(), q.data_ptr(), 0, 0, ncm.F16, 5, 0, 2, 4, 2, 64, cu_q.data_ptr(), cu_k.data_ptr())
    assert bool((out[:4] == 0).all()) and bool((out[4] == 7).all())


def test_prompt_in_a_graph(ncm, cuda):
    """Captured once, replayed with other lengths of the same total."""
    q, k, v = inputs([600], [600], 8, 2, 128, "bf16", seed=7)
    cu, out, s, g = int32([0, 200, 600]), torch.zeros_like(q), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        attend(ncm, q, k, v, cu, cu, "bf16", True, out=out, stream=s.cuda_stream)
    for first in (200, 0, 1, 599):
        cu.copy_(int32([0, first, 600]))
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        check(q, k, v, out, [first, 600 - first], [first, 600 - first], "bf16", True)
