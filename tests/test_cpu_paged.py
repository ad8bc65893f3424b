"""Refusals of the paged cache's calls: decided from the arguments, before any CUDA call."""
import ctypes

import pytest

pytestmark = pytest.mark.cpu

P = 1 << 20   # a non-null, aligned address that is never read


def cache(ncm, **kw):
    a = dict(type=ncm.F16, k_ptr=P, v_ptr=P, pages=10, page_size=16, kv_heads=2, head_dim=64, k_scales_ptr=0,
             v_scales_ptr=0, page_stride=0)
    a.update(kw)
    return ncm.PagedKV(**a)


BAD_CACHES = [dict(type=0), dict(type=14), dict(head_dim=96), dict(head_dim=0), dict(page_size=0), dict(page_size=4),
              dict(page_size=24), dict(page_size=512), dict(kv_heads=0), dict(kv_heads=-1), dict(pages=0),
              dict(pages=1 << 31), dict(page_stride=100), dict(page_stride=2 * 16 * 64 + 8), dict(k_ptr=0), dict(v_ptr=P + 8),
              dict(type=8), dict(type=8, k_scales_ptr=P, v_scales_ptr=P + 2)]


def append(ncm, kv, **kw):
    a = dict(in_type=ncm.F16, q_ptr=P, k_ptr=P, v_ptr=P, q_out_ptr=P, q_out_type=ncm.F16, tokens=4, heads=4, batch=2,
             cu_tokens_ptr=P, lengths_ptr=P, page_table_ptr=P, table_width=5)
    a.update(kw)
    ncm.paged_append(kv, **a)


def attend(ncm, kv, **kw):
    a = dict(out_ptr=P, q_ptr=P, q_type=ncm.F16, batch=2, heads=4, lengths_ptr=P, page_table_ptr=P, table_width=5,
             workspace_ptr=P, workspace_bytes=1 << 30)
    a.update(kw)
    out, q = a.pop("out_ptr"), a.pop("q_ptr")
    ncm.paged_attention(out, q, kv, **a)


def refused(ncm, f, *a, **kw):
    with pytest.raises(ncm.NcmError) as e:
        f(ncm, *a, **kw)
    assert e.value.status == 1, e.value
    return str(e.value)


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_bad_caches(ncm, kw):
    refused(ncm, append, cache(ncm, **kw))
    refused(ncm, attend, cache(ncm, **kw))


@pytest.mark.parametrize("kw", [dict(in_type=8), dict(q_out_type=0), dict(tokens=-1), dict(heads=-1), dict(batch=-1),
                                dict(table_width=0), dict(q_ptr=0), dict(k_ptr=0), dict(v_ptr=0), dict(q_out_ptr=0),
                                dict(lengths_ptr=0), dict(page_table_ptr=0), dict(cu_tokens_ptr=0), dict(k_ptr=P + 2),
                                dict(q_stride=255), dict(k_stride=132), dict(v_stride=-128), dict(rope_style=2),
                                dict(rope_ptr=P, rope_len=0, rope_half=32), dict(rope_ptr=P, rope_len=9, rope_half=34),
                                dict(rope_ptr=P, rope_len=9, rope_half=31), dict(rope_ptr=P + 8, rope_len=9, rope_half=32),
                                dict(rope_ptr=P, rope_len=9, rope_half=16, rope_style=1)])
def test_append_refusals(ncm, kw):
    refused(ncm, append, cache(ncm), **kw)


@pytest.mark.parametrize("kw", [dict(q_type=0), dict(q_type=30), dict(batch=-1), dict(heads=0), dict(heads=5),
                                dict(table_width=0), dict(table_width=1 << 19), dict(out_ptr=0), dict(q_ptr=0),
                                dict(lengths_ptr=0), dict(page_table_ptr=0), dict(workspace_ptr=0), dict(workspace_bytes=64),
                                dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q_stride=100),
                                dict(out_stride=260), dict(out_ptr=P + 2), dict(q_ptr=P + 4), dict(workspace_ptr=P + 4)])
def test_attention_refusals(ncm, kw):
    refused(ncm, attend, cache(ncm), **kw)


def prompt(ncm, **kw):
    a = dict(out_ptr=P, q_ptr=P, k_ptr=P, v_ptr=P, type=ncm.F16, total_q=8, total_k=8, batch=2, heads=4, kv_heads=2,
             head_dim=64, cu_q_ptr=P, cu_k_ptr=P)
    a.update(kw)
    ncm.prompt_attention(**a)


@pytest.mark.parametrize("kw", [dict(type=0), dict(type=8), dict(head_dim=32), dict(head_dim=256), dict(heads=0), dict(kv_heads=0),
                                dict(heads=5), dict(heads=258, kv_heads=2), dict(total_q=-1), dict(total_k=-1), dict(batch=-1),
                                dict(total_q=(1 << 30) + 1), dict(out_ptr=0), dict(q_ptr=0), dict(k_ptr=0), dict(v_ptr=0),
                                dict(cu_q_ptr=0), dict(cu_k_ptr=0), dict(q_ptr=P + 8), dict(out_ptr=P + 2), dict(k_stride=127),
                                dict(q_stride=260), dict(out_stride=-256), dict(v_stride=130), dict(scale=-0.5), dict(scale=float("nan"))])
def test_prompt_refusals(ncm, kw):
    refused(ncm, prompt, **kw)


def test_nothing_to_do_is_no_error(ncm):
    append(ncm, cache(ncm), tokens=0)
    attend(ncm, cache(ncm), batch=0)
    prompt(ncm, total_q=0)
    prompt(ncm, batch=0)


def test_pointers_that_are_not_device_memory_are_refused(ncm):
    host = (ctypes.c_uint8 * 4096)()
    at = (ctypes.addressof(host) + 255) & ~255
    refused(ncm, attend, cache(ncm), out_ptr=at, q_ptr=at)
    refused(ncm, append, cache(ncm), q_ptr=at)


def test_workspace_sizes(ncm):
    assert ncm.paged_attention_workspace(32, 8, 128) > 4096
    assert ncm.paged_attention_workspace(128, 8, 128) > ncm.paged_attention_workspace(32, 8, 128)
    for bad in ((0, 8, 128), (32, 0, 128), (33, 8, 128), (32, 8, 80)):
        with pytest.raises(ncm.NcmError):
            ncm.paged_attention_workspace(*bad)
