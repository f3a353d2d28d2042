"""What the paged-cache operators refuse, through the C ABI and the Python functions, and what they compute on the host.
No GPU: a refused call touches none of its pointers, and none of these calls gets further than its checks."""
import ctypes as C
import math

import pytest
import torch

from vits_amd import _native as N
from vits_amd import ops

P = 1 << 20            # stands for a device address on a 16-byte boundary; never followed
INVALID, WORKSPACE = -1, -4


def refused(rc, word, code=INVALID):
    assert rc == code
    assert word in N.lib.vits_last_error().decode()


PLAN = dict(lengths=P, grow=P + 64, requests=4, table=P + 4096, table_stride=8, width=8, ring=P + 8192, pages=32, cursor=P + 128, page_size=16,
            lengths_out=P + 256, cursor_out=P + 320, row_start=P + 384, row_request=P + 448, row_position=P + 512, row_slot=P + 576, rows=10,
            status=P + 704, stream=0)


@pytest.mark.parametrize("change,word", [
    *[({n: 0}, "null") for n in ("lengths", "grow", "table", "ring", "cursor", "lengths_out", "cursor_out", "row_start", "status",
                                 "row_request", "row_position", "row_slot")],
    (dict(requests=0), "requests"), (dict(requests=65536), "requests"), (dict(rows=-1), "rows"), (dict(rows=(1 << 30) + 1), "rows"),
    (dict(pages=0), "pages"), (dict(pages=(1 << 30) + 1), "pages"), (dict(width=0), "table"), (dict(table_stride=7), "overlap"),
    (dict(page_size=0), "page_size"), (dict(page_size=8), "page_size"), (dict(page_size=24), "page_size"), (dict(page_size=-16), "page_size"),
    (dict(page_size=65552), "page_size"), (dict(lengths_out=P), "in place"), (dict(lengths_out=P + 64), "in place"),
    (dict(cursor_out=P + 128), "in place"), (dict(row_start=P + 60), "in place"), (dict(table=P - 100), "in place"), (dict(ring=P - 100), "in place"),
    (dict(row_slot=P + 516), "two outputs"), (dict(status=P + 8192 + 124), "two outputs"), (dict(lengths_out=P + 4096 + 100), "two outputs"),
])
def test_page_plan_refuses(change, word):
    refused(N.lib.vits_op_page_plan(*{**PLAN, **change}.values()), word)


ROTARY = dict(q=P, q_row=512, q_head=128, out=P + 4096, out_row=512, out_head=128, heads=4, k=P, k_row=256, k_head=128, v=P, v_row=256,
              v_head=128, k_cache=P + (1 << 20), v_cache=P + (2 << 20), page_stride=2 * 16 * 128, pages=9, page_size=16, kv_heads=2, dim=128, dtype=2, position=P,
              slot=P, rows=3, freq=P, pairs=64, scale=1.0, interleaved=0, err_flag=0, stream=0)


@pytest.mark.parametrize("change,word", [
    *[({n: 0}, "null") for n in ("position", "freq", "out", "v", "k_cache", "v_cache", "slot")], (dict(q=0, k=0), "null"),
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(rows=-1), "required"), (dict(dim=1, pairs=1), "required"),
    (dict(dim=258), "required"), (dict(pairs=0), "required"), (dict(pairs=65), "required"), (dict(heads=0), "required"),
    (dict(heads=1025), "required"), (dict(kv_heads=0), "required"), (dict(pages=0), "required"), (dict(page_size=20), "page_size"),
    (dict(page_stride=2 * 16 * 128 - 1), "overlap"), (dict(out=P, out_row=640), "in place"), (dict(out=P, out_row=2048, out_head=512), "in place"),
    (dict(q_row=-1), "strides"), (dict(v_head=-1), "strides"), (dict(out_row=500), "overlap"), (dict(out_head=100), "overlap"), (dict(out_row=0), "overlap"),
    (dict(rows=(1 << 23) + 1), "2^23"), (dict(out=P + 256), "in place"), (dict(k_cache=P + 512), "overlaps"), (dict(v_cache=P + 4096), "overlaps"), (dict(k=P + 4096), "overlaps k or v"),
    (dict(v=P + 5000), "overlaps k or v"), (dict(k_cache=P - (1 << 10)), "overlaps"),
])
def test_rotary_store_refuses(change, word):
    refused(N.lib.vits_op_rotary_store(*{**ROTARY, **change}.values()), word)


M = 1 << 20
ATTEND = dict(q=P, q_row=512, q_head=128, k_cache=P + M, v_cache=P + 2 * M, page_stride=2 * 16 * 128, pages=9, page_size=16, table=P + 3 * M,
              table_stride=8, width=8, requests=3, row_request=P + 4 * M, row_position=P + 5 * M, rows=3, heads=4, kv_heads=2, dim=128, dtype=2,
              scale=0.1, window=0, max_keys=128, out=P + 6 * M, out_row=512, out_head=128, lse=0, err_flag=0, ws=P + 8 * M, ws_bytes=1 << 40,
              stream=0)


@pytest.mark.parametrize("change,word", [
    *[({n: 0}, "null") for n in ("q", "k_cache", "v_cache", "table", "row_request", "row_position", "out")],
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(rows=-1), "required"), (dict(heads=3), "required"), (dict(heads=0), "required"),
    (dict(kv_heads=0), "required"), (dict(heads=2048, kv_heads=2048), "required"), (dict(dim=0), "required"), (dict(dim=48), "required"),
    (dict(dim=288), "required"), (dict(page_size=8), "page_size"), (dict(pages=0), "required"), (dict(width=0), "required"),
    (dict(table_stride=7), "required"), (dict(requests=0), "required"), (dict(window=-1), "required"), (dict(page_stride=100), "overlap"),
    (dict(k_cache=P + M + 8), "16-byte"), (dict(v_cache=P + 2 * M + 2), "16-byte"), (dict(page_stride=2 * 16 * 128 + 4), "16-byte"),
    (dict(out=P), "in place"), (dict(out=P + 1024), "in place"), (dict(out=P + M + 64), "in place"), (dict(out=P + 3 * M), "in place"),
    (dict(lse=P + 2 * M + 64), "in place"), (dict(lse=P + 6 * M + 64), "overlap"), (dict(ws=P + 6 * M), "overlap"), (dict(ws=P), "in place"),
    (dict(q_row=-512), "strides"), (dict(out_head=-128), "strides"), (dict(out_row=0), "strides"), (dict(out_head=64), "strides"),
    (dict(out_row=384), "strides"), (dict(width=1 << 27, table_stride=1 << 27), "2^30"), (dict(rows=(1 << 23) + 1), "2^23"), (dict(q=P + 8), "16-byte"), (dict(q_row=516), "16-byte"), (dict(q_head=132), "16-byte"),
])
def test_paged_attention_refuses(change, word):
    refused(N.lib.vits_op_paged_attention(*{**ATTEND, **change}.values()), word)


def test_paged_attention_workspace():
    size = N.lib.vits_op_paged_attention_workspace_bytes
    for bad in ((-1, 4, 2, 128, 2, 0), (1, 4, 3, 128, 2, 0), (1, 0, 1, 128, 2, 0), (1, 4, 2, 40, 2, 0), (1, 4, 2, 512, 2, 0), (1, 4, 2, 128, 3, 0)):
        assert size(3, *bad) == -1
    need = size(3, 3, 4, 2, 128, 2, 1 << 20)
    assert need > 0 and size(3, 0, 4, 2, 128, 2, 0) >= 0 and size(3, 3, 4, 2, 128, 2, 100) == 0
    assert size(64, 64, 4, 2, 128, 2, 600) == 0 and size(1, 64, 4, 2, 128, 2, 600) > 0               # a row each; a prompt's rows
    if need:
        refused(N.lib.vits_op_paged_attention(*{**ATTEND, "max_keys": 1 << 20, "ws_bytes": need - 1}.values()), "workspace", WORKSPACE)
        refused(N.lib.vits_op_paged_attention(*{**ATTEND, "max_keys": 1 << 20, "ws": 0}.values()), "workspace", WORKSPACE)
        refused(N.lib.vits_op_paged_attention(*{**ATTEND, "max_keys": 1 << 20, "ws": P + 8 * M + 8}.values()), "workspace", WORKSPACE)


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_page_plan_checks_its_tensors():
    """Shapes and types first, so that they can be told here; then that the tensors are on a GPU."""
    pages = ops.new_pages(3, 4, 20, device="cpu")
    good = dict(lengths=pages.lengths, grow=i32(1, 1, 1), table=pages.table, ring=pages.ring, cursor=pages.cursor, page_size=16)
    out = [torch.empty(n, dtype=torch.int64 if i in (1, 5) else torch.int32) for i, n in enumerate((3, 2, 4, 5, 5, 5, 1))]
    with pytest.raises(ValueError, match="GPU"):
        ops.page_plan(**good, rows=4)
    with pytest.raises(ValueError, match="GPU"):
        ops.page_plan(**good, out=out)
    with pytest.raises(ValueError, match="rows or out"):
        ops.page_plan(**good)
    with pytest.raises(ValueError, match="seven"):
        ops.page_plan(**good, out=out[:6])
    for name, bad in (("lengths", pages.lengths.long()), ("grow", i32(1, 1)), ("table", pages.table[:2]), ("table", pages.table.t()),
                      ("table", pages.table.long()), ("table", torch.zeros(3, 8, dtype=torch.int32)[:, ::2]), ("ring", pages.ring.long()),
                      ("ring", pages.ring[::2]), ("cursor", pages.cursor.int()), ("cursor", torch.zeros(3, dtype=torch.int64)), ("grow", None)):
        with pytest.raises(ValueError, match=name):
            ops.page_plan(**{**good, name: bad}, rows=4)
    for i, name in enumerate(("lengths", "cursor", "start", "request", "position", "slot", "status")):
        for bad in (out[i].float(), torch.empty(9, dtype=out[i].dtype)):
            with pytest.raises(ValueError, match="out." + name):
                ops.page_plan(**good, rows=5, out=[*out[:i], bad, *out[i + 1:]])
    with pytest.raises(ValueError, match="out.request"):
        ops.page_plan(**good, rows=6, out=out)


def test_rotary_store_checks_its_tensors():
    q, k, v = torch.zeros(4, 4, 64), torch.zeros(4, 2, 64), torch.zeros(4, 2, 64)
    cache = torch.zeros(5, 2, 2, 16, 64)                       # keys and values of a page side by side
    freq = ops.rotary_frequencies(64, device="cpu")
    good = dict(q=q, k=k, v=v, k_cache=cache[:, 0], v_cache=cache[:, 1], position=i32(0, 1, 2, 3), slot=torch.arange(4), freq=freq)
    alone = dict(k=None, v=None, k_cache=None, v_cache=None)
    for change in ({}, alone, {**alone, "slot": None}, dict(q=None), dict(out=torch.zeros(4, 4, 64)), dict(err_flag=i32(0))):
        with pytest.raises(ValueError, match="GPU"):
            ops.rotary_store(**{**good, **change})
    for change, word in ((dict(q=None, **alone), "neither"), (dict(q=None, out=q), "without q"), (dict(v=None), "together"), (dict(k=None), "together"),
                         (dict(slot=None), "together"), (dict(k_cache=None), "together"), (dict(q=q.double()), "fp32"), (dict(q=q[0]), "rows"),
                         (dict(q=q[:3]), "position"), (dict(k=k[:, :1]), "k must"), (dict(v=v.half()), "v must"), (dict(k=k[..., :32]), "k must"),
                         (dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), "q must"), (dict(out=q[:, :2]), "out must"),
                         (dict(out=q.half()), "out must"), (dict(k_cache=cache[:4, 0]), "alike"), (dict(v_cache=cache[:, 1].contiguous()), "alike"),
                         (dict(k_cache=cache[:, 0].half(), v_cache=cache[:, 1].half()), "caches"),
                         (dict(k_cache=cache[:, 0].transpose(1, 2), v_cache=cache[:, 1].transpose(1, 2)), "alike"),
                         (dict(position=torch.arange(4)), "position"), (dict(slot=i32(0, 1, 2, 3)), "slot"), (dict(freq=freq.float()), "freq"),
                         (dict(err_flag=i32(0, 0)), "err_flag")):
        with pytest.raises(ValueError, match=word):
            ops.rotary_store(**{**good, **change})


def test_paged_attention_checks_its_tensors():
    q, cache = torch.zeros(2, 4, 64), torch.zeros(5, 2, 2, 16, 64)
    good = dict(q=q, k_cache=cache[:, 0], v_cache=cache[:, 1], table=torch.zeros(3, 4, dtype=torch.int32), request=i32(0, 1), position=i32(3, 4))
    for change in ({}, dict(out=torch.zeros(2, 4, 64)), dict(lse=torch.zeros(2, 4)), dict(err_flag=i32(0))):
        with pytest.raises(ValueError, match="GPU"):
            ops.paged_attention(**{**good, **change})
    for change, word in ((dict(q=q.half()), "q must"), (dict(q=q[0]), "rows"), (dict(q=q[..., :32]), "q must"), (dict(table=good["table"].long()), "table"),
                         (dict(table=good["table"][0]), "table"), (dict(request=i32(0)), "request"), (dict(position=torch.tensor([3, 4])), "position"),
                         (dict(out=q.double()), "out must"), (dict(out=torch.zeros(2, 4, 32)), "out must"), (dict(lse=torch.zeros(2, 3)), "lse"),
                         (dict(lse=torch.zeros(2, 4, dtype=torch.float64)), "lse"), (dict(k_cache=cache[:, 0, :, :8]), "alike"),
                         (dict(k_cache=cache[:, 0].long(), v_cache=cache[:, 1].long()), "fp32"), (dict(err_flag=torch.zeros(1)), "err_flag")):
        with pytest.raises(ValueError, match=word):
            ops.paged_attention(**{**good, **change})


def test_rotary_frequencies():
    f = ops.rotary_frequencies(8, device="cpu")
    assert f.dtype == torch.float64 and f.tolist() == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-14)
    assert ops.rotary_frequencies(8, factor=4, scaling="linear", device="cpu").tolist() == pytest.approx([x / 4 for x in f.tolist()], rel=1e-14)
    raised = ops.rotary_frequencies(8, factor=4, scaling="base", device="cpu")
    assert raised[0] == 1.0 and float(raised[3]) == pytest.approx(0.001 / 4, rel=1e-12)
    # pairs that turn more than 32 times in 4096 positions stay, those that turn less than once are divided, those between lie between
    plain = ops.rotary_frequencies(128, device="cpu")
    ramp = ops.rotary_frequencies(128, factor=8, scaling="ramp", device="cpu")
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(ramp[turns > 32], plain[turns > 32])
    assert torch.allclose(ramp[turns < 1], plain[turns < 1] / 8, rtol=1e-14)
    between = (turns > 1) & (turns < 32)
    assert between.any() and bool(((ramp < plain) & (ramp > plain / 8))[between].all())
    assert ops.rotary_frequencies(2, factor=3, scaling="base", device="cpu").tolist() == [1.0]
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, base=1.0),
                dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, scaling="ramp", fast=1.0, slow=1.0), dict(rotary_dim=8, factor=math.nan)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**bad, device="cpu")


def test_gradients_are_refused_not_dropped():
    q, cache, v = torch.zeros(2, 4, 64), torch.zeros(5, 2, 2, 16, 64), torch.zeros(2, 2, 64)
    at = dict(position=i32(3, 4))
    attention = dict(q=q, k_cache=cache[:, 0], v_cache=cache[:, 1], table=torch.zeros(3, 4, dtype=torch.int32), request=i32(0, 1), **at)
    rotary = dict(q=q, k=v, v=v, k_cache=cache[:, 0], v_cache=cache[:, 1], slot=torch.arange(2), freq=ops.rotary_frequencies(64, device="cpu"), **at)
    for call, good, names in ((ops.paged_attention, attention, ("q", "k_cache")), (ops.rotary_store, rotary, ("q", "k", "v"))):
        for name in names:
            asks = {**good, name: good[name].detach().clone(memory_format=torch.preserve_format).requires_grad_()}
            if name == "k_cache":
                asks = {**good, name: cache.clone().requires_grad_()[:, 0]}
            with pytest.raises(ValueError, match="gradient"):
                call(**asks)
            with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
                call(**asks)


def test_strides_of_single_dimensions_say_nothing():
    """One page, one key-value head, one request: views whose stride there is any number are taken (up to the check for a GPU)."""
    def single(shape, stride):
        return torch.zeros(4096 * 4).as_strided(shape, stride)
    q, at = torch.zeros(2, 4, 64), i32(3, 4)
    for shape, stride in (((1, 2, 16, 64), (0, 1024, 64, 1)), ((3, 1, 16, 64), (1024, 64, 64, 1)), ((1, 1, 16, 64), (7, 5, 64, 1))):
        k, v = single(shape, stride), single(shape, stride)
        for table in (torch.zeros(1, 3, dtype=torch.int32), torch.zeros(3, 1, dtype=torch.int32).t()):
            with pytest.raises(ValueError, match="GPU"):
                ops.paged_attention(q, k, v, table, i32(0, 0), at)
