"""Memory that the paged-cache operators would read and write, or write twice, in one launch: refused, on the host, before anything runs.
No GPU: a refused call touches none of its pointers."""
import pytest

from vits_amd import _native as N

P, M = 1 << 24, 1 << 20          # P stands for a device address on a 16-byte boundary; never followed
INVALID = -1
SIZE, DIM = 2, 128               # bf16
HEAD = DIM * SIZE


def refused(rc, word):
    assert rc == INVALID
    assert word in N.lib.vits_last_error().decode()


# q, k and v of a row beside each other (4 + 2 + 2 heads), q turned in place
FUSED = dict(q=P, q_row=8 * DIM, q_head=DIM, out=P, out_row=8 * DIM, out_head=DIM, heads=4, k=P + 4 * HEAD, k_row=8 * DIM, k_head=DIM, v=P + 6 * HEAD,
             v_row=8 * DIM, v_head=DIM, k_cache=P + M, v_cache=P + 2 * M, page_stride=2 * 16 * DIM, pages=9, page_size=16, kv_heads=2, dim=DIM, dtype=2,
             position=P + 3 * M, slot=P + 4 * M, rows=3, freq=P + 5 * M, pairs=64, scale=1.0, interleaved=0, err_flag=P + 6 * M, stream=0)
ROW = 8 * HEAD
# each head's query, key and value beside each other
PER_HEAD = {**FUSED, "kv_heads": 4, "page_stride": 4 * 16 * DIM, "k": P + HEAD, "v": P + 2 * HEAD,
            **{n: 3 * DIM for n in ("q_head", "out_head", "k_head", "v_head")}, **{n: 12 * DIM for n in ("q_row", "out_row", "k_row", "v_row")}}


@pytest.mark.parametrize("base,change", [
    (FUSED, dict(k=P)), (FUSED, dict(v=P)), (FUSED, dict(k=P + 2 * HEAD)), (FUSED, dict(v=P + 3 * HEAD)), (FUSED, dict(v=P + 4 * HEAD - 2)),
    (FUSED, dict(k=P + ROW)), (FUSED, dict(k=P + 2 * ROW + HEAD)), (FUSED, dict(k=P + 7 * HEAD)),             # another row's queries
    (FUSED, dict(k=P - ROW + 3 * HEAD)), (FUSED, dict(k_row=4 * DIM)), (FUSED, dict(v_row=0, v=P + 2 * ROW)), (FUSED, dict(k_head=3 * DIM, v_head=3 * DIM, v=P + 3 * HEAD)),
    (PER_HEAD, dict(k=P)), (PER_HEAD, dict(k=P + HEAD - 2)), (PER_HEAD, dict(v=P + 3 * HEAD)), (PER_HEAD, dict(v=P + 2 * HEAD + 2)),
    (PER_HEAD, dict(k_head=2 * DIM)), ({**FUSED, "rows": 1}, dict(k=P + 3 * HEAD)), ({**FUSED, "rows": 1}, dict(k=P - HEAD)),
])
def test_in_place_rotation_of_shared_rows(base, change):
    refused(N.lib.vits_op_rotary_store(*{**base, **change}.values()), "k or v")


BODY = 2 * 16 * DIM * SIZE       # bytes of a page
PAIRED = {**FUSED, "page_stride": 2 * 2 * 16 * DIM, "v_cache": P + M + BODY}                            # [pages][2][...]


@pytest.mark.parametrize("base,at", [(FUSED, 0), (FUSED, BODY - 2), (FUSED, 2 - BODY), (FUSED, 8 * BODY), (FUSED, 9 * BODY - 2), (PAIRED, 0), (PAIRED, BODY - 2),
                                     (PAIRED, BODY + 2), (PAIRED, 2 * BODY), (PAIRED, -16 * BODY), (PAIRED, 8 * BODY + 16), (PAIRED, 17 * BODY - 2)])
def test_a_cache_over_the_other(base, at):
    refused(N.lib.vits_op_rotary_store(*{**base, "v_cache": P + M + at}.values()), "caches overlap")


@pytest.mark.parametrize("change,word", [
    (dict(position=P + 2 * HEAD), "out"), (dict(slot=P + ROW), "out"), (dict(freq=P + 64), "out"), (dict(err_flag=P + 3 * HEAD), "err_flag"),
    (dict(position=P + M + 64), "cache"), (dict(slot=P + 2 * M - 8), "cache"), (dict(freq=P + 2 * M + 128), "cache"), (dict(err_flag=P + M + 4), "err_flag"),
    (dict(err_flag=P + 3 * M + 8), "err_flag"), (dict(err_flag=P + 4 * M + 20), "err_flag"), (dict(err_flag=P + 5 * M + 508), "err_flag"),
    (dict(err_flag=P + 4 * HEAD), "err_flag"), (dict(err_flag=P + 7 * HEAD), "err_flag"),
    (dict(q=0, out=0, position=P + M), "cache"), (dict(k=0, v=0, k_cache=0, v_cache=0, slot=0, position=P), "out"),
    (dict(k=0, v=0, k_cache=0, v_cache=0, freq=P + 8), "out"), (dict(k=0, v=0, k_cache=0, v_cache=0, err_flag=P + 8), "err_flag"),
    (dict(slot=P + 2 * M + 9 * BODY - 8), "cache"),
])
def test_rotary_store_over_its_rows_numbers(change, word):
    refused(N.lib.vits_op_rotary_store(*{**FUSED, **change}.values()), word)


ATTEND = dict(q=P, q_row=512, q_head=128, k_cache=P + M, v_cache=P + 2 * M, page_stride=2 * 16 * 128, pages=9, page_size=16, table=P + 3 * M,
              table_stride=8, width=8, requests=3, row_request=P + 4 * M, row_position=P + 5 * M, rows=3, heads=4, kv_heads=2, dim=128, dtype=2,
              scale=0.1, window=0, max_keys=128, out=P + 6 * M, out_row=512, out_head=128, lse=P + 7 * M, err_flag=P + 8 * M, ws=P + 9 * M, ws_bytes=1 << 20,
              stream=0)


@pytest.mark.parametrize("at", [P + 8, P + M, P + 2 * M + 400, P + 3 * M + 4, P + 4 * M + 8, P + 5 * M, P + 6 * M + 12, P + 7 * M + 44, P + 9 * M + 16])
def test_paged_attention_err_flag_over_another_tensor(at):
    refused(N.lib.vits_op_paged_attention(*{**ATTEND, "err_flag": at}.values()), "err_flag")
