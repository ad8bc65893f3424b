"""The batched serving operators as they are used together, their calls in a fresh process's
first graph, and their refusal of pointers that are not device memory."""
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_paged import DT, U, Cache, attend64 as attend_one, ids, int32, rope_table, rotated64
from test_gpu_prompt import attend64 as attend_all, starts

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Server:
    """One attention layer of a batch: rows of q, k, v come in, the cache and the outputs follow."""

    def __init__(self, ncm, kind, qkind, style, heads, kvh, hd, page, prompts, steps, seed):
        self.ncm, self.kind, self.qkind, self.style = ncm, kind, qkind, style
        self.heads, self.kvh, self.hd, self.prompts = heads, kvh, hd, prompts
        self.c = Cache(ncm, kind, kvh, hd, page, [n + steps for n in prompts], seed=seed)
        self.rope = rope_table(max(prompts) + steps, hd // 2, hd)
        self.space = torch.zeros(ncm.paged_attention_workspace(heads, kvh, hd), dtype=torch.uint8, device="cuda")
        self.err, self.lengths = int32([0]), int32(prompts)
        self.q = self.out = None

    def append(self, rows, cu, stream=0):
        n, wide, es = rows.shape[0], rows.shape[1] * self.hd, rows.element_size()
        self.ncm.paged_append(self.c.kv, ids(self.ncm)[self.qkind], rows.data_ptr(), rows.data_ptr() + es * self.heads * self.hd,
                              rows.data_ptr() + es * (self.heads + self.kvh) * self.hd, self.q.data_ptr(), ids(self.ncm)[self.qkind],
                              n, self.heads, len(self.prompts), cu.data_ptr() if cu is not None else 0, self.lengths.data_ptr(),
                              self.c.table.data_ptr(), self.c.width, rope_ptr=self.rope.data_ptr(), rope_len=self.rope.shape[0],
                              rope_half=self.hd // 2, rope_style=self.ncm.ROPE_PAIRS if self.style == "pairs" else self.ncm.ROPE_HALVES,
                              q_stride=wide, k_stride=wide, v_stride=wide, err_ptr=self.err.data_ptr(), stream=stream)

    def decode(self, stream=0):
        self.ncm.paged_attention(self.out.data_ptr(), self.q.data_ptr(), self.c.kv, ids(self.ncm)[self.qkind], len(self.prompts), self.heads,
                                 self.lengths.data_ptr(), self.c.table.data_ptr(), self.c.width, self.space.data_ptr(), self.space.numel(),
                                 err_ptr=self.err.data_ptr(), stream=stream)


@pytest.mark.parametrize("kind,qkind,style", [("bf16", "bf16", "pairs"), ("f16", "f16", "halves"), ("q8_0", "bf16", "pairs"), ("q8_0", "f16", "halves")])
def test_prompts_then_steps(ncm, cuda, kind, qkind, style):
    """Prompts: append, attention over them; then steps, captured once: append, attention over the
    cache.  Every stage against 64 bits: the rotated queries, the prompts' outputs on the rotated
    rows that the calls were given, the steps' outputs on what the cache holds."""
    heads, kvh, hd, prompts, steps = 8, 2, 128, [37, 1, 300, 129], 4
    s = Server(ncm, kind, qkind, style, heads, kvh, hd, 16, prompts, steps, seed=7)
    g, n = s.c.g, sum(prompts)
    rows = torch.randn((n, heads + 2 * kvh, hd), generator=g, device="cuda").to(DT[qkind])
    s.q = torch.zeros((n, heads, hd), dtype=DT[qkind], device="cuda")
    cu, at = int32(starts(prompts)), starts(prompts)
    s.append(rows, cu)
    pos = torch.cat([torch.arange(m) for m in prompts]).cuda()
    y, m = rotated64(rows[:, :heads + kvh].double(), s.rope[pos], style, hd // 2)
    assert bool(((s.q.double() - y[:, :heads]).abs() <= U[qkind] * y[:, :heads].abs() + 2.0 ** -22 * m[:, :heads] + 2.0 ** -25).all())
    # the prompts' own attention, over the fresh keys (rotated in the inputs' type) and values
    keys = y[:, heads:].to(DT[qkind]).contiguous()
    values = rows[:, heads + kvh:].contiguous()
    out = torch.zeros_like(s.q)
    ncm.prompt_attention(out.data_ptr(), s.q.data_ptr(), keys.data_ptr(), values.data_ptr(), ids(ncm)[qkind], n, n, len(prompts), heads,
                         kvh, hd, cu.data_ptr(), cu.data_ptr(), err_ptr=s.err.data_ptr())
    for i in range(len(prompts)):
        a, b = at[i], at[i + 1]
        ref, tol = attend_all(s.q[a:b], keys[a:b], values[a:b], hd ** -0.5, 0, qkind)
        assert bool(((out[a:b].double() - ref).abs() <= tol).all())
    # steps
    step = torch.zeros((len(prompts), heads + 2 * kvh, hd), dtype=DT[qkind], device="cuda")
    s.q, s.out = (torch.zeros((len(prompts), heads, hd), dtype=DT[qkind], device="cuda") for _ in range(2))
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        s.append(step, None, stream.cuda_stream)
        s.decode(stream.cuda_stream)
    for i in range(steps):
        s.lengths += 1
        step.copy_(torch.randn(step.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for b, p in enumerate(prompts):
            k = p + i + 1
            ref, tol = attend_one(s.q[b], s.c.rows("k", b, k), s.c.rows("v", b, k), hd ** -0.5, qkind, hd, s.c.rows("v_scales", b, k))
            assert bool(((s.out[b].double() - ref).abs() <= tol).all()), (i, b)
    assert s.err.item() == 0


FIRST = """
import sys, torch
sys.path.insert(0, sys.argv[1]); sys.path.insert(0, sys.argv[1] + "/tests")
import nanocamelid_b200 as ncm
heads, kvh, hd = 8, 2, 64
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
k, v = (torch.zeros((8, kvh, 16, hd), dtype=torch.float16, device="cuda") for _ in range(2))
kv = ncm.PagedKV(ncm.F16, k.data_ptr(), v.data_ptr(), 8, 16, kvh, hd)
rows = torch.randn((20, heads + 2 * kvh, hd), device="cuda").half()
q, out, dec = (torch.zeros((20, heads, hd), dtype=torch.float16, device="cuda") for _ in range(3))
cu, lengths, table, one = i32([0, 20]), i32([20]), i32([[3, 1]]), i32([0, 20])
space = torch.zeros(ncm.paged_attention_workspace(heads, kvh, hd), dtype=torch.uint8, device="cuda")
w, es = (heads + 2 * kvh) * hd, 2
def calls(s):
    ncm.paged_append(kv, ncm.F16, rows.data_ptr(), rows.data_ptr() + es * heads * hd, rows.data_ptr() + es * (heads + kvh) * hd, q.data_ptr(),
                     ncm.F16, 20, heads, 1, cu.data_ptr(), lengths.data_ptr(), table.data_ptr(), 2, q_stride=w, k_stride=w, v_stride=w, stream=s)
    ncm.prompt_attention(out.data_ptr(), q.data_ptr(), rows.data_ptr() + es * heads * hd, rows.data_ptr() + es * (heads + kvh) * hd, ncm.F16, 20, 20,
                         1, heads, kvh, hd, cu.data_ptr(), one.data_ptr(), k_stride=w, v_stride=w, stream=s)
    ncm.paged_attention(dec.data_ptr(), q[19:].data_ptr(), kv, ncm.F16, 1, heads, lengths.data_ptr(), table.data_ptr(), 2, space.data_ptr(),
                        space.numel(), stream=s)
g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
torch.cuda.synchronize()
with torch.cuda.graph(g, stream=s):
    calls(s.cuda_stream)
g.replay(); torch.cuda.synchronize()
first = [x.clone() for x in (q, out, dec)]
calls(0); torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(first, (q, out, dec)))
# the last row of the prompt's attention is the decode step's: two kernels, each within 2^-9 of the row's size
assert float((out[19].float() - dec[0].float()).abs().max()) <= 2.0 ** -9 * float(rows[:, heads + kvh:].abs().max())
print("ok")
"""


def test_first_calls_of_a_process_inside_a_capture(ncm, cuda):
    r = subprocess.run([sys.executable, "-c", FIRST, ROOT], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr


def test_host_pointers_are_refused(ncm, cuda):
    """Each pointer in turn in host memory (pinned, so that the driver knows it)."""
    host = torch.zeros(1 << 16, dtype=torch.uint8).pin_memory()
    dev = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    d, h = dev.data_ptr(), host.data_ptr()

    def refused(f):
        with pytest.raises(ncm.NcmError) as e:
            f()
        assert e.value.status == 1

    kv = ncm.PagedKV(ncm.F16, d, d, 4, 16, 1, 64)
    base = dict(in_type=ncm.F16, q_ptr=d, k_ptr=d, v_ptr=d, q_out_ptr=d, q_out_type=ncm.F16, tokens=1, heads=1, batch=1, cu_tokens_ptr=d,
                lengths_ptr=d, page_table_ptr=d, table_width=1, rope_ptr=d, rope_len=1, rope_half=32, err_ptr=d)
    for name in [k for k in base if k.endswith("_ptr")]:
        refused(lambda: ncm.paged_append(kv, **{**base, name: h}))
    base = dict(q_type=ncm.F16, batch=1, heads=1, lengths_ptr=d, page_table_ptr=d, table_width=1, workspace_ptr=d, workspace_bytes=1 << 30, err_ptr=d)
    for name in [k for k in base if k.endswith("_ptr")]:
        refused(lambda: ncm.paged_attention(d, d, kv, **{**base, name: h}))
    refused(lambda: ncm.paged_attention(h, d, kv, **base))
    refused(lambda: ncm.paged_attention(d, h, kv, **base))
    for field in ("k", "v", "k_scales", "v_scales"):
        bad = ncm.PagedKV(ncm.Q8_0, d, d, 4, 16, 1, 64, d, d)
        setattr(bad, field, h)
        refused(lambda: ncm.paged_attention(d, d, bad, **base))
    base = dict(out_ptr=d, q_ptr=d, k_ptr=d, v_ptr=d, type=ncm.F16, total_q=1, total_k=1, batch=1, heads=1, kv_heads=1, head_dim=64, cu_q_ptr=d,
                cu_k_ptr=d, err_ptr=d)
    for name in [k for k in base if k.endswith("_ptr")]:
        refused(lambda: ncm.prompt_attention(**{**base, name: h}))


def test_two_streams_at_once(ncm, cuda):
    """The same calls on two streams, a workspace each, agree with themselves alone."""
    heads, kvh, hd = 16, 2, 128
    c = Cache(ncm, "bf16", kvh, hd, 32, [20000, 700], seed=3).fill()
    q = torch.randn((2, heads, hd), generator=c.g, device="cuda").bfloat16()
    lengths, size = int32([20000, 700]), ncm.paged_attention_workspace(heads, kvh, hd)
    p, k, v = (torch.randn((3000, n, hd), generator=c.g, device="cuda").bfloat16() for n in (heads, kvh, kvh))
    cu = int32([0, 1000, 3000])

    def calls(out, big, space, s):
        ncm.paged_attention(out.data_ptr(), q.data_ptr(), c.kv, ncm.BF16, 2, heads, lengths.data_ptr(), c.table.data_ptr(), c.width,
                            space.data_ptr(), size, stream=s)
        ncm.prompt_attention(big.data_ptr(), p.data_ptr(), k.data_ptr(), v.data_ptr(), ncm.BF16, 3000, 3000, 2, heads, kvh, hd, cu.data_ptr(),
                             cu.data_ptr(), stream=s)

    outs = [(torch.zeros_like(q), torch.zeros_like(p), torch.zeros(size, dtype=torch.uint8, device="cuda")) for _ in range(3)]
    calls(*outs[0], 0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for o, s in zip(outs[1:], streams):
            calls(*o, s.cuda_stream)
    torch.cuda.synchronize()
    for o in outs[1:]:
        assert torch.equal(o[0], outs[0][0]) and torch.equal(o[1], outs[0][1])
