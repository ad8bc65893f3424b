"""Which check refuses a call of the batched serving operators: the status alone does not tell, since
without a GPU the check of the pointers refuses whatever the others let pass."""
import ctypes

import pytest

from test_cpu_paged import P, append, attend, cache, prompt

pytestmark = pytest.mark.cpu


def reason(ncm, f, *a, **kw):
    with pytest.raises(ncm.NcmError) as e:
        f(ncm, *a, **kw)
    assert e.value.status == 1, e.value
    return str(e.value)


TYPE, SIZE, ROWS, NULL = "type must be", "sizes", "16-byte aligned and at least a token apart", "null pointer"


@pytest.mark.parametrize("kw,why", [
    (dict(type=0), "cache " + TYPE), (dict(type=14), "cache " + TYPE), (dict(head_dim=96), "head_dim must"), (dict(head_dim=0), "head_dim must"),
    (dict(page_size=0), "page_size must"), (dict(page_size=4), "page_size must"), (dict(page_size=24), "page_size must"),
    (dict(page_size=512), "page_size must"), (dict(kv_heads=0), "kv_heads must"), (dict(kv_heads=-1), "kv_heads must"),
    (dict(kv_heads=1025), "kv_heads must"), (dict(pages=0), "pages must"), (dict(pages=-1), "pages must"), (dict(pages=1 << 31), "pages must"),
    (dict(page_stride=100), "page_stride must"), (dict(page_stride=2 * 16 * 64 - 16), "page_stride must"),
    (dict(page_stride=2 * 16 * 64 + 8), "page_stride must"), (dict(page_stride=(1 << 38) + 16), "page_stride must"),
    (dict(k_ptr=0), "k and v must"), (dict(v_ptr=0), "k and v must"), (dict(k_ptr=P + 4), "k and v must"), (dict(v_ptr=P + 8), "k and v must"),
    (dict(type=8), "scales"), (dict(type=8, k_scales_ptr=P), "scales"), (dict(type=8, v_scales_ptr=P), "scales"),
    (dict(type=8, k_scales_ptr=P, v_scales_ptr=P + 2), "scales"), (dict(type=8, k_scales_ptr=P + 8, v_scales_ptr=P), "scales")])
def test_caches(ncm, kw, why):
    assert why in reason(ncm, append, cache(ncm, **kw))
    assert why in reason(ncm, attend, cache(ncm, **kw))


@pytest.mark.parametrize("kw,why", [
    (dict(in_type=8), "in_" + TYPE), (dict(in_type=-1), "in_" + TYPE), (dict(q_out_type=0), "q_out_" + TYPE), (dict(q_out_type=8), "q_out_" + TYPE),
    (dict(tokens=-1), SIZE), (dict(heads=-1), SIZE), (dict(heads=4097), SIZE), (dict(batch=-1), SIZE), (dict(batch=0), SIZE),
    (dict(table_width=0), SIZE), (dict(table_width=-1), SIZE), (dict(table_width=(1 << 22) + 1), SIZE),
    (dict(q_ptr=0), NULL), (dict(k_ptr=0), NULL), (dict(v_ptr=0), NULL), (dict(q_out_ptr=0), NULL), (dict(lengths_ptr=0), NULL),
    (dict(page_table_ptr=0), NULL), (dict(cu_tokens_ptr=0), "without cu_tokens"), (dict(q_ptr=P + 8), ROWS), (dict(k_ptr=P + 2), ROWS),
    (dict(v_ptr=P + 4), ROWS), (dict(q_stride=255), ROWS), (dict(q_stride=248), ROWS), (dict(k_stride=132), ROWS), (dict(v_stride=-128), ROWS),
    (dict(v_stride=(1 << 40) + 8), ROWS), (dict(q_out_ptr=P + 8), "q_out must be"), (dict(rope_style=2), "rope_style"), (dict(rope_style=-1), "rope_style"),
    (dict(rope_ptr=P, rope_len=0, rope_half=32), "rope_len"), (dict(rope_ptr=P, rope_len=9, rope_half=34), "rope_half"),
    (dict(rope_ptr=P, rope_len=9, rope_half=0), "rope_half"), (dict(rope_ptr=P, rope_len=9, rope_half=31), "rope_half"),
    (dict(rope_ptr=P + 8, rope_len=9, rope_half=32), "16-byte"), (dict(rope_ptr=P, rope_len=9, rope_half=16, rope_style=1), "whole head")])
def test_append(ncm, kw, why):
    assert why in reason(ncm, append, cache(ncm), **kw)


@pytest.mark.parametrize("kw,why", [
    (dict(q_type=0), "q_" + TYPE), (dict(q_type=8), "q_" + TYPE), (dict(q_type=30), "one type"), (dict(batch=-1), SIZE), (dict(heads=0), SIZE),
    (dict(heads=-4), SIZE), (dict(heads=5), SIZE), (dict(heads=65538), SIZE), (dict(table_width=-1), SIZE), (dict(table_width=0), "2^22"),
    (dict(table_width=(1 << 18) + 1), "2^22"), (dict(table_width=0x7fffffff), "2^22"), (dict(out_ptr=0), NULL), (dict(q_ptr=0), NULL),
    (dict(lengths_ptr=0), NULL), (dict(page_table_ptr=0), NULL), (dict(workspace_ptr=0), NULL), (dict(workspace_bytes=0), "workspace smaller"),
    (dict(scale=-1.0), "scale must"), (dict(scale=float("nan")), "scale must"), (dict(scale=float("inf")), "scale must"),
    (dict(q_stride=100), ROWS), (dict(q_stride=-256), ROWS), (dict(out_stride=260), ROWS), (dict(out_stride=248), ROWS), (dict(out_ptr=P + 2), ROWS),
    (dict(q_ptr=P + 4), ROWS), (dict(workspace_ptr=P + 4), ROWS), (dict(q_stride=(1 << 40) + 8), ROWS)])
def test_attention(ncm, kw, why):
    assert why in reason(ncm, attend, cache(ncm), **kw)


def test_workspace_border(ncm):
    size = ncm.paged_attention_workspace(4, 2, 64)
    assert "workspace smaller" in reason(ncm, attend, cache(ncm), workspace_bytes=size - 1)
    assert "workspace" not in reason(ncm, attend, cache(ncm), workspace_bytes=size)


@pytest.mark.parametrize("kw,why", [
    (dict(type=0), TYPE), (dict(type=8), TYPE), (dict(head_dim=32), "head_dim must"), (dict(head_dim=256), "head_dim must"), (dict(heads=0), "heads must"),
    (dict(kv_heads=0), "heads must"), (dict(heads=5), "heads must"), (dict(heads=258, kv_heads=2), "heads must"), (dict(heads=2050, kv_heads=1025), "heads must"),
    (dict(total_q=-1), SIZE), (dict(total_k=-1), SIZE), (dict(batch=-1), SIZE), (dict(total_q=(1 << 30) + 1), SIZE), (dict(total_k=(1 << 30) + 1), SIZE),
    (dict(out_ptr=0), NULL), (dict(q_ptr=0), NULL), (dict(k_ptr=0), NULL), (dict(v_ptr=0), NULL), (dict(cu_q_ptr=0), NULL), (dict(cu_k_ptr=0), NULL),
    (dict(q_ptr=P + 8), ROWS), (dict(k_ptr=P + 8), ROWS), (dict(v_ptr=P + 4), ROWS), (dict(out_ptr=P + 2), ROWS), (dict(k_stride=127), ROWS),
    (dict(q_stride=260), ROWS), (dict(q_stride=248), ROWS), (dict(out_stride=-256), ROWS), (dict(v_stride=130), ROWS), (dict(v_stride=(1 << 38) + 8), ROWS),
    (dict(scale=-0.5), "scale must"), (dict(scale=float("nan")), "scale must"), (dict(scale=float("inf")), "scale must")])
def test_prompt(ncm, kw, why):
    assert why in reason(ncm, prompt, **kw)


POINTERS = ("no CUDA device", "a pointer the driver does not know", "not a device pointer")


def test_sound_arguments_reach_the_check_of_the_pointers(ncm):
    """The arguments that the refusals above are variations of: only their made-up addresses are wrong."""
    q8 = dict(type=8, k_scales_ptr=P, v_scales_ptr=P)
    for kw in (dict(), dict(head_dim=128), dict(page_size=8), dict(page_size=256), dict(page_stride=2 * 16 * 64 + 16), q8):
        for f in (append, attend):
            assert reason(ncm, f, cache(ncm, **kw)).split(": ", 1)[1] in POINTERS
    for kw in (dict(q_stride=264), dict(rope_ptr=P, rope_len=9, rope_half=32), dict(rope_ptr=P, rope_len=9, rope_half=32, rope_style=1),
               dict(cu_tokens_ptr=0, tokens=2), dict(heads=0, q_ptr=0, q_out_ptr=0)):
        assert reason(ncm, append, cache(ncm), **kw).split(": ", 1)[1] in POINTERS
    for kw in (dict(), dict(total_k=0, k_ptr=0, v_ptr=0), dict(type=30), dict(scale=2.0), dict(heads=256, kv_heads=2)):
        assert reason(ncm, prompt, **kw).split(": ", 1)[1] in POINTERS


def test_host_memory(ncm):
    host = (ctypes.c_uint8 * 4096)()
    at = (ctypes.addressof(host) + 255) & ~255
    for text in (reason(ncm, attend, cache(ncm), out_ptr=at), reason(ncm, append, cache(ncm), q_ptr=at), reason(ncm, prompt, k_ptr=at)):
        assert text.split(": ", 1)[1] in POINTERS


@pytest.mark.parametrize("off", [1, 2, 3])
def test_int_arrays_off_their_alignment(ncm, off):
    """They are read as ints: an odd address would be a misaligned access on the device."""
    for name in ("cu_tokens_ptr", "lengths_ptr", "page_table_ptr", "err_ptr"):
        assert "4-byte aligned" in reason(ncm, append, cache(ncm), **{name: P + off})
    for name in ("lengths_ptr", "page_table_ptr", "err_ptr"):
        assert "4-byte aligned" in reason(ncm, attend, cache(ncm), **{name: P + off})
    for name in ("cu_q_ptr", "cu_k_ptr", "err_ptr"):
        assert "4-byte aligned" in reason(ncm, prompt, **{name: P + off})


def test_scale_that_overflows_with_the_logarithm(ncm):
    """The kernels take the scale times log2(e), which is infinite from 2.36e38 on."""
    assert "scale must" in reason(ncm, attend, cache(ncm), scale=2.5e38)
    assert "scale must" in reason(ncm, prompt, scale=2.5e38)
    assert "scale" not in reason(ncm, attend, cache(ncm), scale=1.9e38) and "scale" not in reason(ncm, prompt, scale=1.9e38)
