"""The paged-cache operators on the GPU where a call is legal and its data is not what one expects.  Values against 64 bits, with the
bounds that test_gpu_paged.py derives."""
import math

import pytest
import torch

from test_gpu_paged import TYPES, Cache, attend_by_hand, gpu_i32, rows_q

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    from vits_amd import ops
    return ops


@pytest.mark.parametrize("copies,max_keys", [(80, 32), (1, 32), (1, 10 ** 9)])       # a wave a unit, a block a unit, equal pieces
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_attention_of_pages_that_are_none(ops, dtype, copies, max_keys):
    """A row whose every page lies outside the cache sees nothing and gives 0, beside rows of the same request that see a page; a row
    whose pages are there and whose scores are all -inf has no value, whatever other pages are missing."""
    t, page, window, bad = TYPES[dtype], 16, 16, (-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1)
    cache = Cache(t, [32] * (6 * copies), 2, 64, page, seed=31)
    heads, table = 6, cache.table.clone()
    request, position, want = [], [], []                  # want: the first key that counts, None for nothing, "nan" for no value
    for c in range(copies):
        s = 6 * c
        for at, p, w in ((s, 15, None), (s + 1, 31, None), (s + 2, 15, None), (s + 2, 31, 16), (s + 2, 20, 16), (s + 3, 31, "nan"), (s + 4, 20, "nan"),
                         (s + 5, 31, 16)):
            request.append(at)
            position.append(p)
            want.append(w)
        table[s, 0], table[s + 1, 1], table[s + 2, 0], table[s + 4, 0] = bad[c % 4], bad[(c + 1) % 4], bad[(c + 2) % 4], bad[(c + 3) % 4]
        for at in (s + 3, s + 4):
            cache.k_cache[cache.table[at, 1]] = -math.inf
    q = rows_q(cache, len(request), heads, 64, t)
    for r, w in enumerate(want):
        if w == "nan":
            q[r] = 1.0
    flag, lse, out = gpu_i32([0]), torch.full((len(request), heads), 4.0, device="cuda"), torch.full_like(q, 4.0)
    ops.paged_attention(q, cache.k_cache, cache.v_cache, table, gpu_i32(request), gpu_i32(position), window=window, max_keys=max_keys, out=out, lse=lse,
                        err_flag=flag)
    assert flag.item() == 1
    out, lse = out.double().cpu(), lse.double().cpu()
    for r, (s, p, w) in enumerate(zip(request, position, want)):
        if w == "nan":
            assert bool(torch.isnan(out[r]).all()) and bool((lse[r] == -math.inf).all()), r
        elif w is None:
            assert bool((out[r] == 0).all()) and bool((lse[r] == -math.inf).all()), (r, out[r])
        else:
            ref, ref_lse, tol, tol_lse = attend_by_hand(q[r], cache.k[s][w:], cache.v[s][w:], p - w, 1 / 8, window)
            assert bool(((out[r] - ref).abs() <= tol).all()) and bool(((lse[r] - ref_lse).abs() <= tol_lse).all()), r


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_attention_of_missing_pages_over_many_blocks(ops, dtype):
    """The same where a row's keys are cut into pieces that several blocks hold."""
    t, n, far = TYPES[dtype], 20000, 10 ** 6
    cache = Cache(t, [n, n, n], 1, 64, 16, seed=32)
    table = cache.table.clone()
    table[0] = -1
    table[1, :-1] = cache.pages
    cache.k_cache[cache.table[2].long()] = -math.inf
    q = rows_q(cache, 4, 4, 64, t)
    q[2] = 1.0
    for request, position in (([0, 1, 2, -1], [n - 1] * 4), ([0, 1, 2, 0], [n - 1] * 3 + [far])):
        lse, out, flag = torch.full((4, 4), 4.0, device="cuda"), torch.full_like(q, 4.0), gpu_i32([0])
        ops.paged_attention(q, cache.k_cache, cache.v_cache, table, gpu_i32(request), gpu_i32(position), out=out, lse=lse, err_flag=flag)
        assert flag.item() == 1
        out, lse = out.double().cpu(), lse.double().cpu()
        assert bool((out[0] == 0).all() and (lse[0] == -math.inf).all())
        ref, ref_lse, tol, tol_lse = attend_by_hand(q[1], cache.k[1][n - 16:], cache.v[1][n - 16:], 15, 1 / 8, 0)
        assert bool(((out[1] - ref).abs() <= tol).all()) and bool(((lse[1] - ref_lse).abs() <= tol_lse).all())
        assert bool(torch.isnan(out[2]).all() and (lse[2] == -math.inf).all())
        assert bool((out[3] == (4.0 if request[3] < 0 else 0.0)).all())


@pytest.mark.parametrize("max_keys", [32, 10 ** 9])
def test_attention_of_a_position_beyond_the_table(ops, max_keys):
    """What the table holds of its window counts, and the flag says that there was more."""
    t = torch.bfloat16
    cache = Cache(t, [64, 64, 64], 2, 64, 16, seed=33)
    q = rows_q(cache, 3, 4, 64, t)
    position, window = [70, 64 + 19, 2 ** 31 - 1], 20
    for w, low in ((0, [0, 0, 0]), (window, [51, 64, 64])):
        flag, lse = gpu_i32([0]), torch.empty(3, 4, device="cuda")
        out = ops.paged_attention(q, cache.k_cache, cache.v_cache, cache.table, gpu_i32([0, 1, 2]), gpu_i32(position), window=w, max_keys=max_keys, lse=lse,
                                  err_flag=flag).double().cpu()
        assert flag.item() == 1
        for r in range(3):
            ref, ref_lse, tol, tol_lse = attend_by_hand(q[r], cache.k[r][low[r]:], cache.v[r][low[r]:], 63 - low[r], 1 / 8, 0)
            assert bool(((out[r] - ref).abs() <= tol).all()), (w, r)
            assert bool(torch.equal(lse[r].double().cpu(), ref_lse)) if low[r] == 64 else bool(((lse[r].double().cpu() - ref_lse).abs() <= tol_lse).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("layout", ["heads of a row", "each head", "one row for all"])
def test_rotary_in_place_beside_keys(ops, dtype, layout):
    """q turned in place with k and v in the same memory, between its rows or its heads: as from tensors of their own."""
    t, rows, heads, dim = TYPES[dtype], 50, 4, 64
    gen = torch.Generator(device="cuda").manual_seed(41)
    if layout == "each head":
        x = torch.randn(rows, heads, 3, dim, generator=gen, device="cuda").to(t)
        q, k, v = x.unbind(2)
    else:
        x = torch.randn(rows, heads + 4, dim, generator=gen, device="cuda").to(t)
        q, k, v = x[:, :heads], x[:, heads:heads + 2], x[:, heads + 2:]
        if layout == "one row for all":
            k, v = k[7:8].expand(rows, -1, -1), v[49:].expand(rows, -1, -1)
    own = [y.contiguous() for y in (q, k, v)]
    caches = [torch.zeros(4, k.shape[1], 16, dim, dtype=t, device="cuda") for _ in range(4)]
    position, slot, freq = torch.arange(rows, dtype=torch.int32, device="cuda") * 3, torch.randperm(64, generator=gen, device="cuda")[:rows], ops.rotary_frequencies(dim)
    want = ops.rotary_store(*own, caches[0], caches[1], position, slot, freq)
    got = ops.rotary_store(q, k, v, caches[2], caches[3], position, slot, freq, out=q)
    assert got is q and torch.equal(q, want) and torch.equal(k, own[1]) and torch.equal(v, own[2])
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


def test_what_is_written_counts_as_written(ops):
    """Autograd learns of in-place writes by a tensor's version: a cache or an output that a recorded product has saved and a call then
    overwrites makes its backward an error, not a wrong gradient."""
    t = torch.float32
    gen = torch.Generator(device="cuda").manual_seed(42)
    pages = ops.new_pages(2, 4, 8)
    grow = gpu_i32([3, 2])
    plan = ops.page_plan(pages.lengths, grow, pages.table, pages.ring, pages.cursor, 16, rows=6)
    written = [pages.table, pages.ring, *plan]
    before = [x._version for x in written]
    read = [pages.lengths, grow, pages.cursor]
    kept = [x._version for x in read]
    assert ops.page_plan(pages.lengths, grow, pages.table, pages.ring, pages.cursor, 16, out=plan) is plan
    assert all(x._version > n for x, n in zip(written, before)) and [x._version for x in read] == kept

    q, k, v = (torch.randn(6, h, 32, generator=gen, device="cuda") for h in (4, 2, 2))
    both = torch.zeros(8, 2, 2, 16, 32, device="cuda")
    out, lse, flag = torch.zeros_like(q), torch.zeros(6, 4, device="cuda"), gpu_i32([0])
    freq = ops.rotary_frequencies(32)
    store = lambda: ops.rotary_store(q, k, v, both[:, 0], both[:, 1], plan.position, plan.slot, freq, out=out, err_flag=flag)      # noqa: E731
    attend = lambda: ops.paged_attention(q, both[:, 0], both[:, 1], pages.table, plan.request, plan.position, out=out, lse=lse, err_flag=flag)  # noqa: E731
    for call, written, read in ((store, (both, out, flag), (q, k, v, plan.slot, freq)), (attend, (out, lse, flag), (q, both, pages.table))):
        before, kept = [x._version for x in written], [x._version for x in read]
        call()
        assert all(x._version > n for x, n in zip(written, before)) and [x._version for x in read] == kept
    weight = torch.ones_like(both, requires_grad=True)
    loss = (weight * both).sum()
    with torch.no_grad():
        store()
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    with torch.inference_mode():                          # tensors without a version
        caches = [torch.zeros(8, 2, 16, 32, dtype=t, device="cuda") for _ in range(2)]
        ops.rotary_store(q, k, v, *caches, plan.position, plan.slot, freq)
    got = ops.rotary_store(q, k, v, *caches, plan.position, plan.slot, freq)      # an inference tensor outside that mode, as before
    assert torch.equal(caches[0], both[:, 0]) and got.shape == q.shape


def two_term_bounds(t):
    """Of a weight held in two terms of type t, the second of which is what the first leaves of it: each is off by half a step of what it
    holds, so by 2^-22 of the weight in fp16 and 2^-16 in bf16.  fp16 holds nothing below 2^-24, where half a step is 2^-25: the largest
    weight is at least 2^11 there, so that is 2^-36 of it."""
    return {torch.float32: (0.0, 0.0), torch.float16: (2.0 ** -22, 2.0 ** -36), torch.bfloat16: (2.0 ** -16, 0.0)}[t]


def cancelling(t, keys, rows, dim, seed):
    """Rows whose weighted values nearly cancel: the sum is some 2^-9 of its terms, so its own rounding hides nothing of theirs.  Scores are
    products of one channel each (the others are 0), at most 1.5; the last key takes away what the others sum up to."""
    gen = torch.Generator().manual_seed(seed)
    q = torch.zeros(rows, 1, dim)
    q[:, 0, 0] = 1.0
    k = torch.zeros(rows, keys, dim)
    k[:, :, 0] = torch.rand(rows, keys, generator=gen) * 3 - 1.5
    k = k.to(t)
    v = torch.randn(rows, keys, dim, generator=gen).to(t)
    weight = torch.softmax(k[:, :, 0].double(), 1)
    v[:, -1] = (-(weight[:, :-1, None] * v[:, :-1].double()).sum(1) / weight[:, -1:]).to(t)
    return q.to(t), k, v


@pytest.mark.parametrize("max_keys", [32, 10 ** 9])
@pytest.mark.parametrize("keys", [3, 32])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_attention_weights_in_two_terms(ops, dtype, keys, max_keys):
    """The weights enter the second product as exactly as two terms hold them; one alone is found out (planted in the oracle)."""
    t, rows, dim = TYPES[dtype], 24, 64
    q, k, v = cancelling(t, keys, rows, dim, seed=keys)
    cache = Cache(t, [0] * rows, 1, dim, 16, seed=51, width=2, spare=2 * rows)
    cache.table.copy_(torch.arange(2 * rows, dtype=torch.int32, device="cuda").view(rows, 2))
    for r in range(rows):
        for at in range(keys):
            cache.k_cache[2 * r + at // 16, 0, at % 16] = k[r, at].cuda()
            cache.v_cache[2 * r + at // 16, 0, at % 16] = v[r, at].cuda()
    out = ops.paged_attention(q.cuda(), cache.k_cache, cache.v_cache, cache.table, gpu_i32(list(range(rows))), gpu_i32([keys - 1] * rows), scale=1.0,
                              max_keys=max_keys).double().cpu()
    score, values = k[:, :, 0].double(), v.double()
    weight = torch.softmax(score, 1)
    ref = torch.einsum("rn,rnd->rd", weight, values)
    size, most = torch.einsum("rn,rnd->rd", weight, values.abs()), weight.amax(1)[:, None] * values.abs().sum(1)
    held, least = two_term_bounds(t)
    # a score is one product of two values of type t and zeros, exact in fp32; times log2 e and less the maximum: three roundings of at most
    # 2 * 1.5 * log2 e < 8 (with the 11 that fp16 adds: 16), 2^-24 each, and the exponential's own 2^-23: below 2^-18.  Sums of at most 32 terms
    # in fp32, twice, and their quotient: 66 * 2^-24.
    tol = ref.abs() * (torch.finfo(t).eps / 2) + size * (2 * 2.0 ** -18 + 66 * 2.0 ** -24 + held) + least * most
    if t == torch.float16:
        tol = tol + 2.0 ** -25
    assert bool(((out[:, 0] - ref).abs() <= tol).all()), float(((out[:, 0] - ref).abs() / tol).max())
    if t != torch.float32:
        w = torch.exp(score - score.amax(1, keepdim=True))
        one = torch.einsum("rn,rnd->rd", w.to(t).double(), values) / w.sum(1, keepdim=True)
        assert bool(((one - ref).abs() > tol).any(1).float().mean() > 0.5)                # most rows would tell


def test_the_documented_example_runs(ops):
    """The lines of the module's docstring, with a model of one layer."""
    import textwrap
    code = textwrap.dedent("\n".join(x for x in ops.__doc__.splitlines() if x.startswith("    ")))
    assert "page_plan" in code and "paged_attention" in code
    kv_heads, dim, R = 2, 64, 96
    gen = torch.Generator(device="cuda").manual_seed(61)
    q, k, v = (torch.randn(R, h, dim, generator=gen, device="cuda").to(torch.bfloat16) for h in (4, kv_heads, kv_heads))
    names = dict(ops=ops, torch=torch, kv_heads=kv_heads, dim=dim, R=R, q=q, k=k, v=v, grow=torch.ones(64, dtype=torch.int32, device="cuda"))
    exec(code, names)
    assert names["lengths"].tolist() == [1] * 64 and names["plan"].status.item() == 0
    # one token each: it sees itself alone
    assert torch.equal(names["o"][:64], v[:64].repeat_interleave(2, 1)) and not names["o"][64:].any()


def definition(q, k, v, scale):
    """Softmax attention of one row as its formula has it, in 64 bits, infinities and all: q [heads, dim], k and v [keys, kv_heads, dim]."""
    group = q.shape[0] // k.shape[1]
    q, k, v = q.double().cpu(), k.double().cpu().repeat_interleave(group, 1), v.double().cpu().repeat_interleave(group, 1)
    score = torch.stack([(q * x).sum(-1) for x in k]) * scale                                            # [keys, heads]
    weight = torch.softmax(score, 0)
    return torch.stack([(weight[:, h, None] * v[:, h]).sum(0) for h in range(q.shape[0])]), torch.logsumexp(score, 0)


FORMS = [(80, 1, 32), (1, 2, 32), (1, 2, 10 ** 9)]          # copies of the rows, key-value heads, max_keys: a wave a unit, a block, equal pieces


@pytest.mark.parametrize("copies,hk,max_keys", FORMS)
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_attention_of_infinite_values_that_are_seen(ops, dtype, copies, hk, max_keys):
    """A weight times an infinity is that infinity; the two of them together, or a NaN, are NaN; the other channels keep their values.
    Rows alone and beside rows of the same request that do not see it."""
    t = TYPES[dtype]
    cache = Cache(t, [32, 32, 32, 20] * copies, hk, 64, 16, seed=71)
    heads = 3 * hk
    inf = math.inf
    for s in range(4 * copies):
        for at, channel, x in ((17, 3, inf), (17, 9, -inf), (4, 40, inf), (17, 40, -inf), (18, 63, math.nan)):
            if s % 4 != 1:
                cache.v[s][at, :, channel] = x
                cache.v_cache[cache.table[s, at // 16], :, at % 16, channel] = x
    request = [s for c in range(copies) for s in (4 * c, 4 * c + 1, 4 * c + 2, 4 * c + 2, 4 * c + 2, 4 * c + 3)]
    position = [31, 31, 16, 17, 30, 19] * copies
    q = rows_q(cache, len(request), heads, 64, t, gain=1.0)
    lse = torch.empty(len(request), heads, device="cuda")
    out = ops.paged_attention(q, cache.k_cache, cache.v_cache, cache.table, gpu_i32(request), gpu_i32(position), max_keys=max_keys, lse=lse).double().cpu()
    for r, (s, p) in enumerate(zip(request, position)):
        if r >= 12 and r % 31:                             # (the oracle takes its time)
            continue
        ref, ref_lse = definition(q[r], cache.k[s][:p + 1], cache.v[s][:p + 1], 1 / 8)
        wild = ~torch.isfinite(ref)
        assert bool(wild.any()) == (s % 4 != 1 and p > 3)
        assert torch.equal(out[r][wild].nan_to_num(7.0, 8.0, 9.0), ref[wild].nan_to_num(7.0, 8.0, 9.0)), (r, out[r][wild], ref[wild])
        v = cache.v[s].clone()
        v[~torch.isfinite(v)] = 0.0                        # for the bounds of the channels that have a value
        near, _, tol, tol_lse = attend_by_hand(q[r], cache.k[s], v, p, 1 / 8, 0)
        assert bool(((out[r] - near).abs() <= tol)[~wild].all()), r
        assert bool(((lse[r].double().cpu() - ref_lse).abs() <= tol_lse).all())


@pytest.mark.parametrize("copies,hk,max_keys", FORMS)
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_attention_of_infinitely_high_scores(ops, dtype, copies, hk, max_keys):
    """A score of +inf: the row has no value (inf / inf), and the log of its sum is +inf; with a NaN beside it that is NaN too."""
    t = TYPES[dtype]
    cache = Cache(t, [32, 32, 32] * copies, hk, 64, 16, seed=72)
    for s in range(3 * copies):
        if s % 3 != 2:
            cache.k_cache[cache.table[s, 1], :, 5] = math.inf
        if s % 3 == 1:
            cache.k_cache[cache.table[s, 0], :, 2] = math.nan
    request = [s for c in range(copies) for s in (3 * c, 3 * c + 1, 3 * c + 2, 3 * c, 3 * c)]
    position = [31, 31, 31, 20, 21] * copies
    q = rows_q(cache, len(request), 3 * hk, 64, t, gain=1.0).abs()
    lse = torch.empty(len(request), 3 * hk, device="cuda")
    out = ops.paged_attention(q, cache.k_cache, cache.v_cache, cache.table, gpu_i32(request), gpu_i32(position), max_keys=max_keys, lse=lse).double().cpu()
    for r, kind in enumerate(["inf", "nan", "", "", "inf"] * copies):
        if kind:
            assert bool(torch.isnan(out[r]).all()) and bool((lse[r] == math.inf).all() if kind == "inf" else torch.isnan(lse[r]).all()), (r, lse[r])
        else:
            ref, ref_lse, tol, tol_lse = attend_by_hand(q[r], cache.k[request[r]], cache.v[request[r]], position[r], 1 / 8, 0)
            assert bool(((out[r] - ref).abs() <= tol).all()) and bool(((lse[r].double().cpu() - ref_lse).abs() <= tol_lse).all()), r


@pytest.mark.parametrize("max_keys", [None, 10 ** 9])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("heads,hk,dim,page", [(1024, 1, 32, 16), (1024, 1024, 32, 16), (1000, 8, 64, 16), (33, 33, 64, 16), (2, 1, 32, 65536), (48, 3, 96, 4096)])
def test_attention_of_the_largest_heads_and_pages(ops, dtype, heads, hk, dim, page, max_keys):
    t = TYPES[dtype]
    cache = Cache(t, [1, 40, 70], hk, dim, page, seed=81)
    request, position = [2, -1, 0, 1, 1, -1, 1, 2, 2, 2], [69, 3, 0, 38, -1, -1, 39, 5, -1, 60]
    q = rows_q(cache, len(request), heads, dim, t)
    lse, out = torch.full((len(request), heads), 4.0, device="cuda"), torch.full_like(q, 4.0)
    ops.paged_attention(q, cache.k_cache, cache.v_cache, cache.table, gpu_i32(request), gpu_i32(position), max_keys=max_keys, out=out, lse=lse)
    out, lse = out.double().cpu(), lse.double().cpu()
    for r, (s, p) in enumerate(zip(request, position)):
        if s < 0:
            assert bool((out[r] == 4.0).all() and (lse[r] == 4.0).all())
        else:
            ref, ref_lse, tol, tol_lse = attend_by_hand(q[r], cache.k[s], cache.v[s], p, 1 / math.sqrt(dim), 0)
            assert bool(((out[r] - ref).abs() <= tol).all()), r
            assert bool((lse[r] == -math.inf).all()) if p < 0 else bool(((lse[r] - ref_lse).abs() <= tol_lse).all())


def test_rows_beyond_32_bits_of_elements(ops):
    """2^19 + 5 rows of 32 heads of 256: 4.3e9 elements of q and of out, few of them live, the last among them."""
    t, rows, heads, dim = torch.bfloat16, (1 << 19) + 5, 32, 256
    cache = Cache(t, [40, 100], 2, dim, 16, seed=82)
    live = [0, 12345, rows - 3, rows - 2, rows - 1]
    q = torch.zeros(rows, heads, dim, dtype=t, device="cuda")
    q[live] = rows_q(cache, len(live), heads, dim, t)
    request, position = torch.full((rows,), -1, dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    request[live], position[live] = gpu_i32([0, 1, 1, 1, 0]), gpu_i32([39, 99, 7, 8, 20])
    out = torch.full_like(q, 4.0)
    ops.paged_attention(q, cache.k_cache, cache.v_cache, cache.table, request, position, max_keys=100, out=out)
    for r in live:
        s, p = int(request[r]), int(position[r])
        ref, _, tol, _ = attend_by_hand(q[r], cache.k[s], cache.v[s], p, 1 / 16, 0)
        assert bool(((out[r].double().cpu() - ref).abs() <= tol).all()), r
    assert bool((out[1] == 4.0).all() and (out[rows - 4] == 4.0).all())
    slot = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    slot[live] = torch.arange(len(live), device="cuda")
    freq, few = ops.rotary_frequencies(dim), torch.tensor(live, device="cuda")
    want = ops.rotary_store(q[few].contiguous(), None, None, None, None, position[few].contiguous(), None, freq)
    ops.rotary_store(q, None, None, None, None, position, slot, freq, out=out)
    assert torch.equal(out[few], want) and bool((out[1] == 4.0).all() and (out[rows - 4] == 4.0).all())


def test_rotary_of_many_rows(ops):
    gen = torch.Generator(device="cuda").manual_seed(83)
    rows = (1 << 23) - 3
    q = torch.randn(rows, 1, 2, generator=gen, device="cuda")
    position = torch.randint(0, 1 << 20, (rows,), generator=gen, dtype=torch.int32, device="cuda")
    freq = ops.rotary_frequencies(2)
    out = ops.rotary_store(q, None, None, None, None, position, None, freq)
    angle = position.double() * freq
    a, b = q[:, 0, 0].double(), q[:, 0, 1].double()
    ref = torch.stack((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), 1)
    bound = ((a.abs() + b.abs()) * 2.0 ** -21 + 2.0 ** -51 * angle * (a.abs() + b.abs()))[:, None] + ref.abs() * 2.0 ** -24
    assert bool(((out[:, 0].double() - ref).abs() <= bound).all())


def test_plan_of_the_farthest_positions(ops):
    """Lengths up to 2^31 - 1 in pages of 65536, and page ids whose slots need 64 bits."""
    page, width, last = 65536, 32768, 2 ** 31 - 1
    pages = 1 << 20
    table = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
    table[0, :] = torch.arange(width, device="cuda")
    ring = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    ring[5] = pages - 1
    cursor = torch.tensor([5, 6], dtype=torch.int64, device="cuda")
    plan = ops.page_plan(gpu_i32([last - 3, 0]), gpu_i32([3, 2]), table, ring, cursor, page, rows=6)
    assert plan.status.item() == 0 and plan.lengths.tolist() == [last, 2] and plan.start.tolist() == [0, 3, 5] and plan.cursor.tolist() == [6, 6]
    assert plan.request.tolist() == [0, 0, 0, 1, 1, -1] and plan.position.tolist() == [last - 3, last - 2, last - 1, 0, 1, -1]
    top = (width - 1) * page
    assert plan.slot.tolist() == [top + 65532, top + 65533, top + 65534, (pages - 1) * page, (pages - 1) * page + 1, -1]
    assert table[1, 0].item() == pages - 1
    plan = ops.page_plan(gpu_i32([last, 0]), gpu_i32([1, 0]), table, ring, cursor, page, rows=6)
    assert plan.status.item() == 1 and plan.slot.eq(-1).all()
