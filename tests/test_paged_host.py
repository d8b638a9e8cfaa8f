"""What the operators of many sequences refuse, before any device work."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from klcquant_amd import _native as nat
from klcquant_amd import ops

FAKE = 0x1000  # never dereferenced: validation fails first


def refused(name, args, status, text):
    with pytest.raises(nat.KlcError) as ei:
        nat.call(name, *args)
    assert ei.value.status == status and text in ei.value.message, ei.value.message


def prompt_args(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, starts=FAKE, sinks=0, out=FAKE, tokens=10, n_seq=2, n_heads=8, n_kv=2, head_dim=64,
             q_stride=512, k_stride=128, v_stride=128, window=0, dtype=nat.DTYPE_BF16, scale=0.125)
    a.update(kw)
    return ops._PROMPT_ARGS.pack(*a.values()), None


@pytest.mark.parametrize("change,status,text", [
    (dict(q=0), nat.KLC_ERR_ARGUMENT, "null pointer"), (dict(starts=0), nat.KLC_ERR_ARGUMENT, "null pointer"),
    (dict(n_heads=9), nat.KLC_ERR_SHAPE, "heads"), (dict(n_kv=0), nat.KLC_ERR_SHAPE, "heads"),
    (dict(head_dim=60), nat.KLC_ERR_SHAPE, "head_dim"), (dict(head_dim=136), nat.KLC_ERR_SHAPE, "head_dim"),
    (dict(head_dim=0), nat.KLC_ERR_SHAPE, "head_dim"), (dict(tokens=0), nat.KLC_ERR_ARGUMENT, "tokens"),
    (dict(n_seq=0), nat.KLC_ERR_ARGUMENT, "sequences"), (dict(tokens=1 << 29), nat.KLC_ERR_ARGUMENT, "tokens"),
    (dict(q_stride=504), nat.KLC_ERR_SHAPE, "strides"), (dict(k_stride=132), nat.KLC_ERR_SHAPE, "strides"),
    (dict(v_stride=64), nat.KLC_ERR_SHAPE, "strides"), (dict(q=0x1008), nat.KLC_ERR_ARGUMENT, "aligned"),
    (dict(window=-1), nat.KLC_ERR_ARGUMENT, "window"), (dict(scale=0.0), nat.KLC_ERR_ARGUMENT, "scale"),
    (dict(scale=float("nan")), nat.KLC_ERR_ARGUMENT, "scale"), (dict(scale=float("inf")), nat.KLC_ERR_ARGUMENT, "scale"),
    (dict(dtype=nat.DTYPE_F32), nat.KLC_ERR_UNSUPPORTED, "dtype")])
def test_prompt_refusals(change, status, text):
    refused("klc_attn_prompt", prompt_args(**change), status, text)


def append_args(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, cos=FAKE, sin=FAKE, positions=FAKE, slots=FAKE, q_out=FAKE, k_out=0, k_pages=FAKE,
             v_pages=FAKE, tokens=10, n_positions=100, n_slots=64, n_heads=8, n_kv=2, head_dim=64, q_stride=512,
             k_stride=128, v_stride=128, kv_dtype=nat.DTYPE_F16)
    a.update(kw)
    return ops._APPEND_ARGS.pack(*a.values()), None


@pytest.mark.parametrize("change,status,text", [
    (dict(cos=0), nat.KLC_ERR_ARGUMENT, "null pointer"), (dict(k_pages=0), nat.KLC_ERR_ARGUMENT, "null pointer"),
    (dict(head_dim=12), nat.KLC_ERR_SHAPE, "head_dim"), (dict(n_heads=0), nat.KLC_ERR_SHAPE, "heads"),
    (dict(tokens=0), nat.KLC_ERR_ARGUMENT, "tokens"), (dict(n_positions=0), nat.KLC_ERR_ARGUMENT, "positions"),
    (dict(n_slots=1 << 31), nat.KLC_ERR_ARGUMENT, "slots"), (dict(k_stride=100), nat.KLC_ERR_SHAPE, "strides"),
    (dict(sin=0x1004), nat.KLC_ERR_ARGUMENT, "aligned"),
    (dict(k_out=0x1008), nat.KLC_ERR_ARGUMENT, "aligned"),
    (dict(kv_dtype=nat.DTYPE_F32), nat.KLC_ERR_UNSUPPORTED, "kv_dtype")])
def test_append_refusals(change, status, text):
    refused("klc_kv_append", append_args(**change), status, text)


@pytest.mark.parametrize("change,text", [(dict(pools=None), "null pointer"), (dict(n_pools=0), "pools"), (dict(n_pages=0), "pages"),
                                         (dict(page_bytes=24), "multiple of 16"), (dict(pools=0x1008), "aligned"),
                                         (dict(src=[0, 8]), "move 1"), (dict(dst=[-1, 2]), "move 0"), (dict(n=-1), "moves"),
                                         (dict(dst=[3, 3]), "another move"), (dict(dst=[4, 0]), "another move")])
def test_copy_refusals(change, text):
    a = dict(pools=FAKE, n_pools=2, n_pages=8, page_bytes=1024, src=[0, 1], dst=[2, 3], n=2, stream=None)
    a.update(change)
    a["src"], a["dst"] = ((ctypes.c_int32 * 2)(*a[x]) for x in ("src", "dst"))
    refused("klc_kv_copy_pages", list(a.values()), nat.KLC_ERR_ARGUMENT, text)


def batch_args(**kw):
    a = dict(q=FAKE, k_pages=FAKE, v_pages=FAKE, tables=FAKE, lengths=FAKE, prefix_table=FAKE, sinks=0, workspace=FAKE,
             out=FAKE, n_seq=4, n_heads=8, n_kv=2, head_dim=64, q_stride=512, n_pages=32, page_size=64, table_width=4,
             prefix_len=100, window=0, kv_dtype=nat.DTYPE_F16, workspace_bytes=1 << 30, scale=0.125)
    a.update(kw)
    return ops._BATCH_ARGS.pack(*a.values()), None


@pytest.mark.parametrize("change,status,text", [
    (dict(lengths=0), nat.KLC_ERR_ARGUMENT, "null pointer"), (dict(workspace=0, prefix_len=3000), nat.KLC_ERR_ARGUMENT, "workspace"),
    (dict(tables=0), nat.KLC_ERR_ARGUMENT, "null table"), (dict(prefix_table=0), nat.KLC_ERR_ARGUMENT, "null table"),
    (dict(page_size=8), nat.KLC_ERR_SHAPE, "power of two"), (dict(page_size=48), nat.KLC_ERR_SHAPE, "power of two"),
    (dict(page_size=8192), nat.KLC_ERR_SHAPE, "power of two"),
    (dict(page_size=4096, n_heads=4096, n_kv=4096, q_stride=4096 * 64), nat.KLC_ERR_SHAPE, "2 GiB"), (dict(n_pages=1 << 26), nat.KLC_ERR_SHAPE, "pages"),
    (dict(table_width=-1), nat.KLC_ERR_SHAPE, "tables"), (dict(n_heads=66, q_stride=66 * 64), nat.KLC_ERR_SHAPE, "group"),
    (dict(head_dim=68), nat.KLC_ERR_SHAPE, "head_dim"), (dict(n_seq=0), nat.KLC_ERR_ARGUMENT, "sequences"),
    (dict(n_seq=70000), nat.KLC_ERR_ARGUMENT, "sequences"), (dict(prefix_len=-1), nat.KLC_ERR_ARGUMENT, "prefix"),
    (dict(window=-3), nat.KLC_ERR_ARGUMENT, "window"), (dict(table_width=1 << 24), nat.KLC_ERR_ARGUMENT, "own tokens"),
    (dict(q_stride=500), nat.KLC_ERR_SHAPE, "stride"), (dict(out=0x1008), nat.KLC_ERR_ARGUMENT, "aligned"),
    (dict(scale=-1.0), nat.KLC_ERR_ARGUMENT, "scale"), (dict(kv_dtype=nat.DTYPE_F32), nat.KLC_ERR_UNSUPPORTED, "kv_dtype"),
    (dict(workspace_bytes=64, prefix_len=3000), nat.KLC_ERR_ARGUMENT, "workspace")])
def test_batch_refusals(change, status, text):
    refused("klc_attn_batch", batch_args(**change), status, text)


def test_batch_workspace_bytes():
    size = lambda *a: nat.call("klc_attn_batch_workspace_bytes", *a)  # noqa: E731
    row = 4 * 64 + 8  # of one part
    for n_seq, prefix, own, window, parts in ((1, 0, 0, 0, 0), (200, 0, 64, 0, 0), (65535, 0, 64, 0, 0), (200, 1000, 2048, 128, 0),
                                              (64, 8192, 704, 0, 2), (1, 0, 1 << 20, 0, 2)):
        got = size(n_seq, 64, 8, 64, prefix, own, window)
        assert got % (n_seq * 64 * row) == 0 and got >= n_seq * 64 * row * parts
    refused("klc_attn_batch_workspace_bytes", (0, 64, 8, 64, 0, 0, 0), nat.KLC_ERR_ARGUMENT, "sequences")
    refused("klc_attn_batch_workspace_bytes", (4, 64, 1, 64, 0, 0, 0), nat.KLC_ERR_SHAPE, "group")


def test_cpu_tensors_are_refused():
    x = torch.zeros((3, 8, 64), dtype=torch.bfloat16)
    kv = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    pages = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)
    index = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.prompt_attention(x, kv, kv, index)
    with pytest.raises(ValueError, match="GPU"):
        ops.batch_attention(x, pages, pages, index[:, None], index)
    with pytest.raises(ValueError, match="GPU"):
        ops.paged_append(x, kv, kv, x, x, index, index, pages, pages)
    with pytest.raises(ValueError, match="GPU"):
        ops.copy_pages(pages[None], [0], [1])
    for call in (lambda: ops.prompt_attention(None, kv, kv, index), lambda: ops.batch_attention([], pages, pages, index, index),
                 lambda: ops.paged_append(np.zeros(3), kv, kv, x, x, index, index, pages, pages)):
        with pytest.raises(TypeError, match="torch.Tensor"):
            call()


@pytest.mark.parametrize("scale,fine", [(2.3e38, True), (2.4e38, False), (3.3e38, False), (1e39, False)])
def test_scales_are_finite_as_the_kernels_hold_them(scale, fine):
    """In powers of two a scale is log2(e) times itself: past 2.36e38 that is infinite, and every score of 0 NaN."""
    for name, args in (("klc_attn_prompt", prompt_args(scale=scale, dtype=nat.DTYPE_F32)),
                       ("klc_attn_batch", batch_args(scale=scale, kv_dtype=nat.DTYPE_F32))):
        # the type is refused behind the scale
        refused(name, args, nat.KLC_ERR_UNSUPPORTED if fine else nat.KLC_ERR_ARGUMENT, "dtype" if fine else "scale")
