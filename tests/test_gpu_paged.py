"""The paged-cache operators on the GPU against plain implementations on the host: whole numbers in Python, values in 64 bits.

Tolerances, set before the first run.  A value rounded to type t is off by at most eps(t) / 2 of itself; below the normal
range of fp16 by 2^-25.
Rotation: cosine and sine carry the rounding of the reduced angle (2^-24 of at most pi / 4), of the function (one unit, 2^-23
of at most 1) and of the scale (2^-24), the two products and their sum 2^-24 each: below 2^-21 of scale * (|a| + |b|).  The
angle itself is a product in 64 bits on both sides, the kernel's one more to count in turns: 2^-51 of it covers the three roundings.
Attention: a score s = scale * q . k of dim products, summed in fp32 in any order, is off by at most es = (dim + 4) * 2^-24 *
scale * sum |q k|.  A weight then is off by the factor 1 + 2 es (its own score and the sum's) + 2^-19 (the exponential
of a difference of up to 2^3 ... 2^6 in fp32, taken as a power of two: the argument's 2^-24 of 64 times ln 2, and the function's 2^-23), the sums
over n keys add n * 2^-24 each, and a weight that is held in 16 bits for the product with v adds half a unit of fp16, 2^-11,
and 2^-25 absolute of a weight of at most 1 (bf16 weights are split in two and lose 2^-16).  All of these scale sum w |v|."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    from vits_amd import ops
    return ops


def half_step(ref, dtype):
    return ref.abs() * (torch.finfo(dtype).eps / 2) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


# ---------------------------------------------------------------------------------------------------------------------
# page plan
# ---------------------------------------------------------------------------------------------------------------------
def plan_by_hand(lengths, grow, table, ring, cursor, page, rows):
    """The plan, request by request, token by token, on Python lists; table and ring are changed."""
    from vits_amd import _native as N
    n, cap, width = len(lengths), len(ring), len(table[0])
    status = 0
    for l, g in zip(lengths, grow):
        if l < 0 or g < -1 or (g > 0 and l + g >= 1 << 31):
            status |= N.PLAN_BAD_LENGTH
        elif -(-(l + max(g, 0)) // page) > width:
            status |= N.PLAN_TABLE_FULL
    good = [(l, g) for l, g in zip(lengths, grow) if not (l < 0 or g < -1 or (g > 0 and l + g >= 1 << 31))]
    fresh = sum(-(-(l + max(g, 0)) // page) - -(-l // page) for l, g in good)
    back = sum(-(-l // page) for l, g in good if g < 0)
    head, tail = cursor
    if head < 0 or tail < head or tail - head > cap or tail - head + back > cap:
        status |= N.PLAN_BAD_RING
    if sum(max(g, 0) for _, g in good) > rows:
        status |= N.PLAN_ROWS_FULL
    if fresh > tail - head:
        status |= N.PLAN_NO_PAGES
    out = dict(lengths=list(lengths), cursor=[head, tail], start=[0] * (n + 1), request=[-1] * rows, position=[-1] * rows, slot=[-1] * rows,
               status=[status])
    if status:
        return out
    row = 0
    for s in range(n):
        out["start"][s] = row
        held = -(-lengths[s] // page)
        if grow[s] < 0:
            for j in range(held):
                ring[tail % cap] = table[s][j]
                tail += 1
            out["lengths"][s] = 0
            continue
        for t in range(lengths[s], lengths[s] + grow[s]):
            if t // page >= held:
                table[s][held] = ring[head % cap]
                head += 1
                held += 1
            out["request"][row], out["position"][row], out["slot"][row] = s, t, table[s][t // page] * page + t % page
            row += 1
        out["lengths"][s] = lengths[s] + grow[s]
    out["start"][n], out["cursor"] = row, [head, tail]
    return out


def plan_state(seed, lengths, page, width, spare, head=None):
    """Tables whose requests hold random distinct pages, and a ring with the rest of them."""
    rng = random.Random(seed)
    need = sum(-(-l // page) for l in lengths if l > 0)
    pages = need + spare
    ids = list(range(pages))
    rng.shuffle(ids)
    table, at = [], 0
    for l in lengths:
        k = -(-l // page) if l > 0 else 0
        table.append(ids[at:at + k][:width] + [-7] * (width - k))
        at += k
    head = rng.randrange(5 * pages + 1) if head is None else head
    ring = [-9] * pages
    for i, p in enumerate(ids[need:]):
        ring[(head + i) % pages] = p
    return table, ring, [head, head + spare]


def gpu_i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check_plan(ops, lengths, grow, page, width, spare, rows, seed=0, head=None, cursor=None, out=None, strided=False):
    table, ring, cur = plan_state(seed, lengths, page, width, spare, head)
    cur = cursor or cur
    dev_table = gpu_i32(table)
    if strided:
        dev_table = torch.nn.functional.pad(dev_table, (0, 5), value=77)[:, :width]
    dev = (gpu_i32(lengths), gpu_i32(grow), dev_table, gpu_i32(ring), torch.tensor(cur, dtype=torch.int64, device="cuda"))
    want = plan_by_hand(lengths, grow, table, ring, cur, page, rows)
    for _ in range(2):                                   # the inputs that are not in place are unchanged: the step can be taken again
        plan = ops.page_plan(*dev, page, rows=rows, out=out)
        for name, values in want.items():
            assert getattr(plan, name).tolist() == values, name
        assert dev[2].tolist() == table
        assert dev[3].tolist() == ring
        assert dev[0].tolist() == lengths and dev[1].tolist() == grow and dev[4].tolist() == cur
    return want


@pytest.mark.parametrize("page", [16, 48, 128])
@pytest.mark.parametrize("requests,longest,prompt", [(1, 1, 1), (1, 5000, 3000), (3, 40, 0), (64, 300, 90), (256, 100, 5), (257, 100, 70),
                                                      (700, 64, 9), (5000, 40, 2)])
def test_plan_of_mixed_steps(ops, page, requests, longest, prompt):
    rng = random.Random(requests * 1000 + page)
    lengths = [rng.choice((0, rng.randint(0, longest), page, page - 1, page + 1)) for _ in range(requests)]
    grow = [rng.choice((-1, 0, 1, 1, 1, rng.randint(0, prompt))) for _ in lengths]
    total = sum(max(g, 0) for g in grow)
    width = max(-(-(l + max(g, 0)) // page) for l, g in zip(lengths, grow)) or 1
    fresh = sum(-(-(l + max(g, 0)) // page) - -(-l // page) for l, g in zip(lengths, grow))
    for pad, spare in ((0, fresh), (13, fresh + 7)):
        want = check_plan(ops, lengths, grow, page, width, spare or 1, total + pad, seed=pad, strided=pad > 0)
        assert want["status"] == [0]


@pytest.mark.parametrize("total", [1023, 1024, 1025, 4096, 70001])
def test_plan_of_prompts_across_blocks(ops, total):
    """Requests that begin, end and lie wholly inside, at and across the borders of a block's rows."""
    rng = random.Random(total)
    grow = []
    while sum(grow) < total:
        grow.append(min(total - sum(grow), rng.choice((1, 2, 0, 511, 1024, rng.randint(1, 3000)))))
    check_plan(ops, [0] * len(grow), grow, 16, -(-max(grow) // 16), sum(-(-g // 16) for g in grow), total + 3)


def test_plan_of_the_most_requests(ops):
    """65535 requests: a thread sums 256 of them, and a block serves 32."""
    rng = random.Random(65535)
    lengths = [rng.randint(0, 70) for _ in range(65535)]
    grow = [rng.choice((-1, 0, 1, 1, 3)) for _ in lengths]
    fresh = sum(-(-(l + max(g, 0)) // 16) - -(-l // 16) for l, g in zip(lengths, grow))
    want = check_plan(ops, lengths, grow, 16, 5, fresh, sum(max(g, 0) for g in grow) + 9)
    assert want["status"] == [0]


def test_plan_without_rows(ops):
    check_plan(ops, [40, 17, 0], [-1, 0, -1], 16, 3, 4, 0)
    check_plan(ops, [40, 17, 0], [-1, 0, -1], 16, 3, 4, 5)


def test_plan_far_cursor(ops):
    check_plan(ops, [5, 100, 33], [30, -1, 1], 16, 8, 9, 40, head=(1 << 40) + 12345)


def test_plan_refuses_on_the_gpu(ops):
    from vits_amd import _native as N
    cases = [
        (dict(lengths=[3, -1], grow=[1, 1]), N.PLAN_BAD_LENGTH), (dict(lengths=[3, 4], grow=[-2, 1]), N.PLAN_BAD_LENGTH),
        (dict(lengths=[3, 4], grow=[1, 2 ** 31 - 1]), N.PLAN_BAD_LENGTH), (dict(lengths=[3, 60], grow=[1, 5]), N.PLAN_TABLE_FULL),
        (dict(lengths=[3, 40], grow=[10, 7], rows=16), N.PLAN_ROWS_FULL), (dict(lengths=[16, 32], grow=[17, 16], spare=2), N.PLAN_NO_PAGES),
        (dict(lengths=[3, 40], grow=[1, 1], cursor=[5, 4]), N.PLAN_BAD_RING | N.PLAN_NO_PAGES * 0),
        (dict(lengths=[3, 40], grow=[1, 1], cursor=[0, 1000]), N.PLAN_BAD_RING), (dict(lengths=[3, 40], grow=[1, 1], cursor=[-3, 1]), N.PLAN_BAD_RING),
        (dict(lengths=[3, 40], grow=[1, -1], cursor=[0, 6]), N.PLAN_BAD_RING),
    ]
    for case, bit in cases:
        want = check_plan(ops, case["lengths"], case["grow"], 16, 4, case.get("spare", 2), case.get("rows", 40), cursor=case.get("cursor"), head=3)
        assert want["status"][0] & bit


@pytest.mark.parametrize("lengths,grow,bits", [([0] * 4, [1 << 30] * 4, "ROWS_FULL"), ([0] * 300, [1 << 30] * 4 + [0] * 296, "ROWS_FULL"),
                                               ([2 ** 31 - 1] * 32, [-1] * 32, "BAD_RING"), ([2 ** 31 - 1] * 512, [-1] * 512, "BAD_RING"),
                                               ([0] * 32, [2 ** 31 - 1] * 32, "NO_PAGES")])
def test_plan_of_sums_beyond_32_bits(ops, lengths, grow, bits):
    """Sums that are a multiple of 2^32: refused, not taken for nothing."""
    from vits_amd import _native as N
    width, rows = 4, 40
    table, ring = [[0] * width for _ in lengths], list(range(6))
    dev = (gpu_i32(lengths), gpu_i32(grow), gpu_i32(table), gpu_i32(ring), torch.tensor([0, 6], dtype=torch.int64, device="cuda"))
    want = plan_by_hand(lengths, grow, table, ring, [0, 6], 16, rows)
    plan = ops.page_plan(*dev, 16, rows=rows)
    assert plan.status.item() & getattr(N, "PLAN_" + bits)
    for name, values in want.items():
        assert getattr(plan, name).tolist() == values, name
    assert dev[2].tolist() == table and dev[3].tolist() == ring


def test_plan_into_unaligned_buffers(ops):
    lengths, grow = [3, 100, 0, 16], [1, 1, 90, 40]
    rows = 137
    def cut(n, dtype):
        return torch.full((n + 3,), 5, dtype=dtype, device="cuda")[1:n + 1]
    i32, i64 = torch.int32, torch.int64
    out = tuple(cut(n, t) for n, t in ((4, i32), (2, i64), (5, i32), (rows, i32), (rows, i32), (rows, i64), (1, i32)))
    check_plan(ops, lengths, grow, 16, 8, 20, rows, out=out)
    for t in out:                                        # and nothing behind them
        assert t._base[0] == 5 and t._base[t.numel() + 1:].eq(5).all()


def test_plan_python_refusals(ops):
    pages = ops.new_pages(3, 4, 20)
    grow = gpu_i32([1, 1, 1])
    good = (pages.lengths, grow, pages.table, pages.ring, pages.cursor, 16)
    for i, bad in ((0, pages.lengths.long()), (1, grow[:2]), (2, pages.table[:2]), (2, pages.table.t()), (3, pages.ring.long()),
                   (4, pages.cursor.int()), (0, pages.lengths.cpu()), (5, 17)):
        args = list(good)
        args[i] = bad
        with pytest.raises((ValueError, RuntimeError)):
            ops.page_plan(*args, rows=4)
    plan = ops.page_plan(*good, rows=4)
    for i in range(7):
        bad = list(plan)
        bad[i] = bad[i][:-1] if i not in (3, 4, 5) else bad[i].float()
        with pytest.raises(ValueError):
            ops.page_plan(*good, rows=4, out=bad)
    with pytest.raises(ValueError, match="seven"):
        ops.page_plan(*good, rows=4, out=plan[:6])
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.page_plan(*good, rows=4, out=plan._replace(lengths=pages.lengths))


# ---------------------------------------------------------------------------------------------------------------------
# rotary rows
# ---------------------------------------------------------------------------------------------------------------------
def rotate_by_hand(x, position, freq, interleaved, scale):
    """The rotation in 64 bits, and how far fp32 arithmetic may be from it."""
    x = x.double().cpu()
    n = 2 * freq.numel()
    angle = position.double().cpu()[:, None] * freq.double().cpu()
    c, s = angle.cos()[:, None, :], angle.sin()[:, None, :]
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., :n // 2], x[..., n // 2:n])
    out, size = x.clone(), torch.zeros_like(x)
    first, second, both = scale * (a * c - b * s), scale * (b * c + a * s), scale * (a.abs() + b.abs()) * (2.0 ** -21 + 2.0 ** -51 * angle.abs()[:, None, :])
    if interleaved:
        out[..., 0:n:2], out[..., 1:n:2], size[..., 0:n:2], size[..., 1:n:2] = first, second, both, both
    else:
        out[..., :n // 2], out[..., n // 2:n], size[..., :n // 2], size[..., n // 2:n] = first, second, both, both
    return out, size


def near_rotation(got, ref, size, dtype):
    assert got.dtype == dtype
    off = (got.double().cpu() - ref).abs()
    assert bool((off <= half_step(ref, dtype) + size).all()), float((off - half_step(ref, dtype) - size).max())


def make_rows(dtype, rows, hq, hk, dim, layout, gen):
    """q, k, v as parts of one tensor, as tensors of their own, or off the 16-byte addresses."""
    if layout == "fused":
        x = torch.randn(rows, hq + 2 * hk, dim, generator=gen, device="cuda").to(dtype)
        return x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    cut = 1 if layout == "odd" else 0
    return tuple(torch.randn(rows * h * dim + cut, generator=gen, device="cuda").to(dtype)[cut:].view(rows, h, dim) for h in (hq, hk, hk))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,hq,hk,dim,rot,layout", [
    (1, 2, 2, 96, 96, "own"), (1, 1, 1, 2, 2, "own"), (7, 8, 2, 64, 64, "fused"), (5, 4, 4, 128, 32, "fused"), (33, 6, 3, 80, 62, "fused"),
    (3, 5, 1, 36, 10, "own"), (9, 4, 2, 128, 128, "odd"), (300, 3, 1, 256, 256, "fused"), (1000, 1, 1, 32, 16, "fused"), (6, 2, 1, 33, 32, "own"),
])
def test_rotary_store(ops, dtype, interleaved, rows, hq, hk, dim, rot, layout):
    t = TYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(rows * 31 + dim)
    q, k, v = make_rows(t, rows, hq, hk, dim, layout, gen)
    page, pages = 16, rows // 16 + 3
    cache = torch.randn(pages, 2, hk, page, dim, generator=gen, device="cuda").to(t)     # keys and values of a page side by side
    before = cache.clone()
    rng = random.Random(rows)
    position = torch.tensor([rng.choice((0, 1, rng.randrange(1000), rng.randrange(2 ** 20), 2 ** 31 - 1)) for _ in range(rows)], dtype=torch.int32, device="cuda")
    slot = torch.randperm(pages * page, generator=gen, device="cuda")[:rows]
    if rows > 4:
        slot[rng.randrange(rows)] = -1
        slot[rows - 1] = -1
    freq = ops.rotary_frequencies(rot)
    scale = 1.25
    out = torch.full((rows, hq, dim), 3.0, dtype=t, device="cuda")
    back = ops.rotary_store(q, k, v, cache[:, 0], cache[:, 1], position, slot, freq, interleaved=interleaved, scale=scale, out=out)
    assert back is out
    live = (slot >= 0).cpu()
    ref, size = rotate_by_hand(q, position, freq, interleaved, scale)
    near_rotation(out[live], ref[live], size[live], t)
    assert torch.equal(out[..., rot:][live], q[..., rot:][live]) and bool((out[~live] == 3.0).all())
    ref, size = rotate_by_hand(k, position, freq, interleaved, scale)
    s = slot[live]
    near_rotation(cache[s // page, 0, :, s % page], ref[live], size[live], t)
    assert torch.equal(cache[s // page, 1, :, s % page], v[live])
    cache[s // page, :, :, s % page] = before[s // page, :, :, s % page]
    assert torch.equal(cache, before)                                                  # no other cell was written


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,hq,hk,dim,rot,layout", [(1, 96, 8, 96, 96, "own"), (2, 64, 8, 192, 182, "odd"), (3, 40, 8, 256, 2, "fused"),
                                                       (300, 5, 5, 34, 22, "odd"), (1100, 32, 8, 64, 54, "fused")])
def test_rotary_store_in_slices(ops, dtype, interleaved, rows, hq, hk, dim, rot, layout):
    """A row's items over several blocks, several rows a block, heads that end beside 16 bytes; in place, with slots outside the
    cache: those rows' queries stay too, and the flag says so."""
    t = TYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(rows + dim)
    q, k, v = make_rows(t, rows, hq, hk, dim, layout, gen)
    page, pages = 32, rows // 32 + 2
    k_cache, v_cache = (torch.randn(pages, hk, page, dim, generator=gen, device="cuda").to(t) for _ in range(2))
    position = torch.randint(0, 2 ** 20, (rows,), generator=gen, dtype=torch.int32, device="cuda")
    slot = torch.randperm(pages * page, generator=gen, device="cuda")[:rows]
    if rows > 1:
        slot[rows // 2] = pages * page
    freq, flag, live = ops.rotary_frequencies(rot), gpu_i32([0]), (slot < pages * page).cpu()
    old, parts = q.clone(), (q, k, v)
    turned = ops.rotary_store(*parts, k_cache, v_cache, position, slot, freq, interleaved=interleaved, out=q, err_flag=flag)
    assert turned is q and flag.item() == (rows > 1)
    ref, size = rotate_by_hand(old, position, freq, interleaved, 1.0)
    near_rotation(q[live], ref[live], size[live], t)
    assert torch.equal(q[..., rot:], old[..., rot:]) and torch.equal(q[~live], old[~live])
    s = slot[live]
    ref, size = rotate_by_hand(k, position, freq, interleaved, 1.0)
    near_rotation(k_cache[s // page, :, s % page], ref[live], size[live], t)
    assert torch.equal(v_cache[s // page, :, s % page], v[live])


def test_rotary_store_many_items(ops):
    """So many that a thread takes several, over ragged heads off the 16-byte addresses: the same bits as for few rows at a time."""
    gen = torch.Generator(device="cuda").manual_seed(31)
    rows, hq, hk, dim, rot, page = 4000, 40, 8, 66, 54, 16
    for t, interleaved in ((torch.float32, False), (torch.bfloat16, True)):
        q, k, v = make_rows(t, rows, hq, hk, dim, "odd", gen)
        caches = [torch.zeros(rows // page, hk, page, dim, dtype=t, device="cuda") for _ in range(4)]
        position = torch.arange(rows, dtype=torch.int32, device="cuda") + 77
        slot = torch.randperm(rows, generator=gen, device="cuda")
        slot[5::7] = -1
        freq = ops.rotary_frequencies(rot)
        out = ops.rotary_store(q, k, v, caches[0], caches[1], position, slot, freq, interleaved=interleaved)
        for i in range(0, rows, 500):
            part = slice(i, i + 500)
            few = ops.rotary_store(q[part], k[part], v[part], caches[2], caches[3], position[part], slot[part], freq, interleaved=interleaved)
            assert torch.equal(few, out[part])
        assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_rotary_parts_alone(ops, dtype):
    """Queries without keys (new, in place, strided out), keys without queries."""
    t = TYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = make_rows(t, 20, 4, 2, 64, "fused", gen)
    position = torch.arange(20, dtype=torch.int32, device="cuda") * 7
    freq = ops.rotary_frequencies(64)
    ref, size = rotate_by_hand(q, position, freq, False, 1.0)
    out = ops.rotary_store(q, None, None, None, None, position, None, freq)
    near_rotation(out, ref, size, t)
    wide = torch.zeros(20, 4, 72, dtype=t, device="cuda")
    ops.rotary_store(q, None, None, None, None, position, None, freq, out=wide[..., 4:68])
    assert torch.equal(wide[..., 4:68], out) and not wide[..., :4].any() and not wide[..., 68:].any()
    k_cache, v_cache = (torch.zeros(2, 2, 16, 64, dtype=t, device="cuda") for _ in range(2))
    slot = torch.arange(20, device="cuda")
    assert ops.rotary_store(None, k, v, k_cache, v_cache, position, slot, freq) is None
    ref, size = rotate_by_hand(k, position, freq, False, 1.0)
    near_rotation(k_cache[slot // 16, :, slot % 16], ref, size, t)
    assert torch.equal(v_cache[slot // 16, :, slot % 16], v)
    slot[3] = -1
    fresh = ops.rotary_store(q, None, None, None, None, position, slot, freq)
    assert not fresh[3].any() and torch.equal(fresh[4:], out[4:])
    ops.rotary_store(q, None, None, None, None, position, None, freq, out=q)
    assert torch.equal(q, out)
    none = q[:0]
    assert ops.rotary_store(none, None, None, None, None, position[:0], None, freq).shape == (0, 4, 64)


def test_rotary_gradient(ops):
    """The gradient is the rotation by the negated frequencies: against the formula's transpose, and against differences."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    for interleaved in (False, True):
        x, g = (torch.randn(6, 2, 32, generator=gen, device="cuda") for _ in range(2))
        position = torch.tensor([0, 1, 5, 999, 123456, 2 ** 30], dtype=torch.int32, device="cuda")
        freq = ops.rotary_frequencies(24)
        call = lambda y, f: ops.rotary_store(y, None, None, None, None, position, None, f, interleaved=interleaved, scale=1.5)  # noqa: E731
        dx = call(g, -freq)
        y = x.double().cpu().requires_grad_()
        n = 24
        angle = position.double().cpu()[:, None] * freq.cpu()
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        a, b = (y[..., 0:n:2], y[..., 1:n:2]) if interleaved else (y[..., :n // 2], y[..., n // 2:n])
        u, w = 1.5 * (a * c - b * s), 1.5 * (b * c + a * s)
        g64 = g.double().cpu()
        gu, gw = (g64[..., 0:n:2], g64[..., 1:n:2]) if interleaved else (g64[..., :n // 2], g64[..., n // 2:n])
        ((u * gu).sum() + (w * gw).sum() + (y[..., n:] * g64[..., n:]).sum()).backward()
        _, size = rotate_by_hand(g, position, freq, interleaved, 1.5)
        near_rotation(dx, y.grad, size, torch.float32)
        # differences: the map is linear, so a step of 1 has no curvature; each of the two sums of 64 products of fp32 values
        # carries 2^-21 of its terms' magnitudes
        d = torch.randn(6, 2, 32, generator=gen, device="cuda")
        slope = ((call(x + d, freq).double() - call(x, freq).double()) * g.double()).sum()
        terms = ((x + d).abs() + x.abs()).double().sum() * 2 * 1.5 * float(g.abs().max())
        assert abs(float(slope - (dx.double() * d.double()).sum())) <= 2.0 ** -20 * float(terms)


def test_rotary_slots_outside_the_cache(ops):
    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = make_rows(torch.float32, 4, 2, 1, 32, "own", gen)
    whole = torch.full((6, 1, 16, 32), 9.0, device="cuda")
    k_cache, v_cache = whole[1:3], whole[3:5]                                           # pages before and behind them are watched
    position, freq = gpu_i32([1, 2, 3, 4]), ops.rotary_frequencies(32)
    flag = gpu_i32([0])
    out = torch.full_like(q, 5.0)
    ops.rotary_store(q, k, v, k_cache, v_cache, position, torch.tensor([31, -1, -2 ** 60, 0], device="cuda"), freq, out=out, err_flag=flag)
    assert flag.item() == 0 and bool((out[1:3] == 5.0).all()) and bool((out[0] != 5.0).any())
    whole.fill_(9.0)
    ops.rotary_store(q, k, v, k_cache, v_cache, position, torch.tensor([32, 2 ** 40, 2 ** 62, 7], device="cuda"), freq, out=out, err_flag=flag)
    assert flag.item() == 1
    assert bool((whole[0] == 9).all() and (whole[2] == 9).all() and (whole[4:] == 9).all())
    assert torch.equal(v_cache[0, :, 7], v[3]) and bool((out[1:3] == 5.0).all())


def test_rotary_python_refusals(ops):
    gen = torch.Generator(device="cuda").manual_seed(6)
    q, k, v = make_rows(torch.bfloat16, 4, 4, 2, 64, "own", gen)
    k_cache, v_cache = (torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    good = dict(q=q, k=k, v=v, k_cache=k_cache, v_cache=v_cache, position=gpu_i32([0, 1, 2, 3]), slot=torch.arange(4, device="cuda"),
                freq=ops.rotary_frequencies(64))
    ops.rotary_store(**good)
    for bad in (dict(q=q.double()), dict(q=q[:3]), dict(k=k[:, :1]), dict(v=v.half()), dict(v=None), dict(k=None), dict(slot=None),
                dict(k_cache=k_cache[..., :32], v_cache=v_cache[..., :32]), dict(k_cache=k_cache.half(), v_cache=v_cache.half()),
                dict(position=good["position"].long()), dict(slot=good["slot"].int()), dict(freq=good["freq"].float()),
                dict(freq=ops.rotary_frequencies(66)), dict(out=q[:, :2]), dict(out=q.transpose(0, 1)), dict(q=None, out=q),
                dict(q=q[1:], out=q[:3], k=None, v=None, k_cache=None, v_cache=None, slot=None, position=good["position"][1:]),
                dict(err_flag=torch.zeros(2, dtype=torch.int32, device="cuda")), dict(slot=good["slot"].cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            ops.rotary_store(**{**good, **bad})


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
class Cache:
    """Requests of given lengths with pages spread over a cache; cells that belong to no token hold `junk`."""

    def __init__(self, dtype, lengths, hk, dim, page, seed, junk=float("nan"), width=None, spare=2):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        need = [-(-n // page) for n in lengths]
        self.lengths, self.page, self.pages = lengths, page, sum(need) + spare
        both = torch.full((self.pages, 2, hk, page, dim), junk, dtype=dtype, device="cuda")
        self.k_cache, self.v_cache = both[:, 0], both[:, 1]
        ids = torch.randperm(self.pages, generator=self.gen, device="cuda").tolist()
        width = width or max(max(need), 1)
        table, self.k, self.v, at = [], [], [], 0
        for n, p in zip(lengths, need):
            mine = ids[at:at + p]
            at += p
            table.append(mine + [-1] * (width - p))
            k, v = (torch.randn(n, hk, dim, generator=self.gen, device="cuda").to(dtype) for _ in range(2))
            for j, pid in enumerate(mine):
                part = slice(j * page, min((j + 1) * page, n))
                both[pid, 0, :, :part.stop - part.start] = k[part].transpose(0, 1)
                both[pid, 1, :, :part.stop - part.start] = v[part].transpose(0, 1)
            self.k.append(k)
            self.v.append(v)
        self.table = gpu_i32(table)


def attend_by_hand(q, k, v, position, scale, window):
    """One row: q [heads, dim], k and v [tokens, kv_heads, dim]; out, lse and the bounds of their errors, in 64 bits."""
    heads, dim = q.shape
    low = max(0, position + 1 - window) if window else 0
    group = heads // k.shape[1]
    dtype = q.dtype
    q, k, v = q.double().cpu(), k[low:position + 1].double().cpu(), v[low:position + 1].double().cpu()
    n = k.shape[0]
    if n == 0:
        return torch.zeros(heads, dim, dtype=torch.float64), torch.full((heads,), -math.inf, dtype=torch.float64), 0.0, 0.0
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)              # [n, heads, dim]
    score = torch.einsum("hd,nhd->hn", q, k) * scale
    weight = torch.softmax(score, 1)
    out = torch.einsum("hn,nhd->hd", weight, v)
    size = torch.einsum("hn,nhd->hd", weight, v.abs())
    es = (dim + 4) * 2.0 ** -24 * abs(scale) * torch.einsum("hd,nhd->hn", q.abs(), k.abs()).amax(1, keepdim=True)
    lse = torch.logsumexp(score, 1)
    held = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -16}[dtype]
    tol = half_step(out, dtype) + size * (2 * es + 2.0 ** -19 + 2 * n * 2.0 ** -24 + held)
    if dtype == torch.float16:                                                         # weights below fp16's normal range
        tol = tol + 2.0 ** -25 * v.abs().sum(0) * torch.exp(score.amax(1) - lse)[:, None]
    return out, lse, tol, es[:, 0] + 2.0 ** -19 + n * 2.0 ** -24 + lse.abs() * 2.0 ** -23


def check_attention(ops, cache, q, request, position, scale=None, window=0, max_keys=None, out=None):
    rows, heads, dim = q.shape
    flag = gpu_i32([0])
    if out is None:
        out = torch.full((rows, heads, dim), 4.0, dtype=q.dtype, device="cuda")
    lse = torch.full((rows, heads), 4.0, device="cuda")
    back = ops.paged_attention(q, cache.k_cache, cache.v_cache, cache.table, gpu_i32(request), gpu_i32(position), scale=scale, window=window,
                               max_keys=max_keys, out=out, lse=lse, err_flag=flag)
    assert back is out and flag.item() == 0
    got, got_lse = out.double().cpu(), lse.double().cpu()
    for r, (s, p) in enumerate(zip(request, position)):
        if s < 0:
            assert bool((got[r] == 4.0).all() and (got_lse[r] == 4.0).all()), r
            continue
        ref, ref_lse, tol, tol_lse = attend_by_hand(q[r], cache.k[s], cache.v[s], p, 1 / math.sqrt(dim) if scale is None else scale, window)
        off = (got[r] - ref).abs()
        assert bool((off <= tol).all()), (r, s, p, float(off.max()), float((off - tol).max()))
        if p < 0:
            assert bool((got_lse[r] == -math.inf).all())
        else:
            assert bool(((got_lse[r] - ref_lse).abs() <= tol_lse).all()), (r, s, p, got_lse[r], ref_lse)
    return got


def rows_q(cache, rows, heads, dim, dtype, gain=1.5):
    return torch.randn(rows, heads, dim, generator=cache.gen, device="cuda").mul_(gain).to(dtype)


@pytest.mark.parametrize("max_keys", [None, 10 ** 9])               # a block a unit, or equal pieces of all the work
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("heads,hk,dim,page", [(2, 2, 96, 16), (8, 2, 128, 32), (5, 1, 64, 48), (16, 1, 32, 16), (17, 1, 64, 16), (24, 2, 160, 16),
                                               (40, 1, 192, 64), (4, 4, 224, 16), (6, 3, 256, 128)])
def test_attention_heads_and_lengths(ops, dtype, heads, hk, dim, page, max_keys):
    """Every length around the borders of tiles and pages, a row that sees nothing, and rows that are none."""
    t = TYPES[dtype]
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300]
    cache = Cache(t, lengths, hk, dim, page, seed=dim + heads)
    request = list(range(len(lengths))) + [-1, 3, -1]
    position = [n - 1 for n in lengths] + [5, -1, -1]
    check_attention(ops, cache, rows_q(cache, len(request), heads, dim, t), request, position, max_keys=max_keys)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attention_of_many_short_rows(ops, dtype, dim):
    """So many units that a wave takes one by itself; every twelfth row against the oracle."""
    t = TYPES[dtype]
    rng = random.Random(dim)
    lengths = [rng.randint(1, 32) for _ in range(540)]
    cache = Cache(t, lengths, 1, dim, 16, seed=dim)
    request = [s if s % 12 != 5 else -1 for s in range(540)]
    position = [n - 1 for n in lengths]
    q = rows_q(cache, 540, 3, dim, t)
    out = torch.full((540, 3, dim), 4.0, dtype=t, device="cuda")
    ops.paged_attention(q, cache.k_cache, cache.v_cache, cache.table, gpu_i32(request), gpu_i32(position), max_keys=32, out=out)
    assert torch.isfinite(out).all()
    for r in range(0, 540, 12):
        ref, _, tol, _ = attend_by_hand(q[r], cache.k[r], cache.v[r], position[r], 1 / math.sqrt(dim), 0)
        assert bool(((out[r].double().cpu() - ref).abs() <= tol).all()), r
        assert bool((out[r + 5] == 4.0).all())
    # the same rows in equal pieces and a block a unit: a wave's sums are in another order
    for rows, keys in ((540, 10 ** 9), (500, 32)):
        other = ops.paged_attention(q[:rows], cache.k_cache, cache.v_cache, cache.table, gpu_i32(request[:rows]), gpu_i32(position[:rows]), max_keys=keys)
        for r in range(0, rows, 12):
            ref, _, tol, _ = attend_by_hand(q[r], cache.k[r], cache.v[r], position[r], 1 / math.sqrt(dim), 0)
            assert bool(((other[r].double().cpu() - ref).abs() <= tol).all()), r


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("heads,hk", [(3, 1), (16, 1), (8, 4)])
def test_attention_of_one_long_row_among_short_ones(ops, dtype, heads, hk):
    """A unit that reaches over most of the pieces beside units that share one."""
    t = TYPES[dtype]
    lengths = [5] * 20 + [30000] + [70] * 19
    cache = Cache(t, lengths, hk, 64, 16, seed=heads)
    check_attention(ops, cache, rows_q(cache, 40, heads, 64, t), list(range(40)), [n - 1 for n in lengths])


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("window", [1, 2, 16, 17, 50, 128, 1000, 5000])
def test_attention_window(ops, dtype, window):
    t = TYPES[dtype]
    cache = Cache(t, [1, 40, 200, 1111], 2, 64, 16, seed=window)
    request = [0, 1, 2, 3, 3, 3, 2, 3]
    position = [0, 39, 199, 1110, 0, 500, 16, -1]
    check_attention(ops, cache, rows_q(cache, 8, 6, 64, t), request, position, window=window)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lengths", [[9000], [5000, 3, 900, 1], [20000, 700]])
@pytest.mark.parametrize("max_keys", [None, 64, 10 ** 9])
def test_attention_long(ops, dtype, lengths, max_keys):
    """Few rows over long lengths, whatever the host believes them to be."""
    t = TYPES[dtype]
    cache = Cache(t, lengths, 2, 128, 16, seed=len(lengths))
    request = list(range(len(lengths)))
    check_attention(ops, cache, rows_q(cache, len(lengths), 8, 128, t), request, [n - 1 for n in lengths], max_keys=max_keys)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("group,window", [(1, 0), (2, 0), (3, 40), (8, 7)])
def test_attention_several_rows_of_a_request(ops, dtype, group, window):
    """A prompt's rows, and drafted tokens: rows of one request beside each other, each with its own end."""
    t = TYPES[dtype]
    cache = Cache(t, [70, 500, 33], 2, 64, 16, seed=group)
    request = [0] * 70 + [1] * 5 + [2] * 3 + [1, 2, 1]
    position = list(range(70)) + [495, 496, 497, 498, 499] + [30, 31, 32] + [5, 0, 499]
    check_attention(ops, cache, rows_q(cache, len(request), 2 * group, 64, t), request, position, window=window)


@pytest.mark.parametrize("rows", [300, 1500])
def test_attention_many_rows(ops, rows):
    rng = random.Random(rows)
    lengths = [rng.randint(1, 90) for _ in range(rows)]
    cache = Cache(torch.bfloat16, lengths, 1, 64, 16, seed=rows)
    request = [s if rng.random() > 0.1 else -1 for s in range(rows)]
    check_attention(ops, cache, rows_q(cache, rows, 2, 64, torch.bfloat16), request, [n - 1 for n in lengths])


@pytest.mark.parametrize("max_keys", [None, 700, 16])
@pytest.mark.parametrize("dtype,heads,hk,window", [("bf16", 8, 2, 0), ("fp16", 3, 3, 50), ("fp32", 16, 1, 0)])
def test_attention_of_prompts(ops, dtype, heads, hk, window, max_keys):
    """Whole prompts row by row, beside a row that comes twice and rows of requests in turn, out of order."""
    cache = Cache(TYPES[dtype], [700, 90], hk, 64, 32, seed=25)
    request = [0] * 700 + [1] * 90 + [0, 0] + [1, 0] * 20
    position = list(range(700)) + list(range(90)) + [411, 411] + [x for i in range(20) for x in (89 - i, 17 * i)]
    check_attention(ops, cache, rows_q(cache, len(request), heads, 64, TYPES[dtype]), request, position, window=window, max_keys=max_keys)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_attention_strides(ops, dtype):
    """Queries as part of a larger tensor, off the 16-byte addresses too, an output with gaps, a negative and a large scale."""
    t = TYPES[dtype]
    cache = Cache(t, [50, 130], 2, 64, 16, seed=1, width=20)
    cache.table = torch.nn.functional.pad(cache.table, (0, 3), value=10 ** 9)[:, :20]
    for cut in (0, 1):
        wide = torch.randn(2, 9, 66, generator=cache.gen, device="cuda").to(t)
        q = wide[:, 2:6, cut:cut + 64]
        buf = torch.full((2, 7, 70), 8.0, dtype=t, device="cuda")
        for scale in (-0.3, 2.0):
            check_attention(ops, cache, q, [1, 0], [129, 49], scale=scale, out=buf[:, 1:5, cut:cut + 64])
        assert bool((buf[:, 0] == 8).all() and (buf[:, 5:] == 8).all() and (buf[..., :cut] == 8).all() and (buf[..., cut + 64:] == 8).all())


@pytest.mark.parametrize("window,max_keys", [(30, None), (0, 10 ** 9)])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_attention_ignores_what_is_not_seen(ops, dtype, window, max_keys):
    """Infinities and NaN behind a row's position, before its window, in its page's unused cells and in other pages change no
    bit of it: also for a row whose neighbour of the same request does see them."""
    t = TYPES[dtype]
    cache = Cache(t, [90, 200], 2, 64, 16, seed=9, junk=0.0)
    q = rows_q(cache, 6, 8, 64, t)
    request, position = gpu_i32([0, 0, 0, 0, 1, 1]), gpu_i32([60, 61, 62, 89, 100, 199])
    args = dict(table=cache.table, request=request, position=position, window=window, max_keys=max_keys)
    clean = ops.paged_attention(q, cache.k_cache, cache.v_cache, **args)
    for junk in (float("nan"), float("inf"), -float("inf")):
        k, v = cache.k_cache.clone(), cache.v_cache.clone()
        def spoil(s, t0, t1):
            for tok in range(t0, t1):
                pid = int(cache.table[s, tok // 16])
                k[pid, :, tok % 16] = junk
                v[pid, :, tok % 16] = junk
        spoil(0, 62, 90)                       # seen by rows 2 and 3 alone
        if window:
            spoil(0, 0, 31)
            spoil(1, 101, 170)
            spoil(1, 0, 71)
        used = set(cache.table.flatten().tolist())
        for pid in range(cache.pages):
            if pid not in used:
                k[pid] = junk
                v[pid] = junk
        got = ops.paged_attention(q, k, v, **args)
        for r in (0, 1, 4, 5):                 # (row 5 sees 101 .. 170 without a window)
            assert torch.equal(got[r], clean[r]), (junk, r)
        assert bool((~torch.isfinite(got[2])).any())


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_attention_infinite_scores(ops, dtype):
    """Keys of -inf scores have no weight while another key has one; where all are -inf, or one is NaN, softmax has no value."""
    t = TYPES[dtype]
    cache = Cache(t, [40, 40, 40, 700], 1, 32, 16, seed=11, junk=0.0)
    q = torch.ones(4, 1, 32, dtype=t, device="cuda")
    k = cache.k_cache
    lowest = -math.inf
    for s, tokens in ((0, range(0, 39)), (1, range(0, 40)), (3, range(0, 650))):
        for tok in tokens:
            k[int(cache.table[s, tok // 16]), :, tok % 16] = lowest
    k[int(cache.table[2, 1]), :, 3] = float("nan")
    lse = torch.zeros(4, 1, device="cuda")
    out = ops.paged_attention(q, k, cache.v_cache, cache.table, gpu_i32([0, 1, 2, 3]), gpu_i32([39, 39, 39, 699]), lse=lse)
    assert torch.equal(out[0, 0], cache.v[0][39, 0])
    assert bool(torch.isnan(out[1]).all()) and lse[1].item() == lowest
    assert bool(torch.isnan(out[2]).all()) and math.isnan(lse[2].item())
    kept = cache.k[3].clone()
    kept[:650] = 0
    ref, _, tol, _ = attend_by_hand(q[3], kept[650:], cache.v[3][650:], 49, 1 / math.sqrt(32), 0)
    assert bool(((out[3].double().cpu() - ref).abs() <= tol).all())


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_attention_large_scores(ops, dtype):
    """Scores far apart: only their differences count, and a dominant key takes all."""
    t = TYPES[dtype]
    cache = Cache(t, [300], 1, 64, 16, seed=12)
    q = rows_q(cache, 1, 4, 64, t, gain=40.0)
    check_attention(ops, cache, q, [0], [299])


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_attention_of_many_small_weights(ops, dtype):
    """A first key of weight 1 and 10^5 more of e^-17.75 = 2^-25.6 each, less than fp16's least number: together they are 2e-3 of
    the sum.  n roundings follow each other in a sum (16 adds of a lane, its column, four waves, 391 blocks: below 450), on
    both sides of the division."""
    t, n, dim = TYPES[dtype], 100000, 32
    cache = Cache(t, [0], 1, dim, 16, seed=22, width=n // 16 + 1, spare=n // 16 + 1)
    cache.table.copy_(torch.randperm(cache.pages, device="cuda").to(torch.int32)[None])
    k, v = torch.zeros(n, 1, dim, dtype=t, device="cuda"), torch.full((n, 1, dim), -1.0, dtype=t, device="cuda")
    k[1:, :, 0] = -17.75
    v[0] = 1.0
    slot = cache.table[0].long()[torch.arange(n, device="cuda") // 16] * 16 + torch.arange(n, device="cuda") % 16
    ops.rotary_store(None, k, v, cache.k_cache, cache.v_cache, torch.zeros(n, dtype=torch.int32, device="cuda"), slot, ops.rotary_frequencies(dim))
    q = torch.zeros(1, 1, dim, dtype=t, device="cuda")
    q[..., 0] = 1.0
    lse = torch.empty(1, 1, device="cuda")
    out = ops.paged_attention(q, cache.k_cache, cache.v_cache, cache.table, gpu_i32([0]), gpu_i32([n - 1]), scale=1.0, lse=lse).double().cpu()
    rest = (n - 1) * math.exp(-17.75)
    ref = torch.full((1, 1, dim), (1 - rest) / (1 + rest), dtype=torch.float64)
    near = 2 * (dim + 4) * 2.0 ** -24 * 17.75 + 2.0 ** -19 + 2 * 450 * 2.0 ** -24 + {"fp32": 0.0, "fp16": 2.0 ** -21, "bf16": 2.0 ** -16}[dtype]
    assert bool(((out - ref).abs() <= half_step(ref, t) + near).all()), (out[0, 0, 0].item(), ref[0, 0, 0].item())
    assert abs(lse.item() - math.log1p(rest)) <= near


def test_attention_ids_outside(ops):
    """Pages outside the cache are left out, requests and positions outside the table not followed; the flag says so."""
    t = torch.bfloat16
    cache = Cache(t, [100, 60], 2, 64, 16, seed=13)
    q = rows_q(cache, 2, 4, 64, t)
    for bad in (-1, cache.pages, 2 ** 31 - 1, -2 ** 31):
        table = cache.table.clone()
        table[0, 2] = bad
        flag = gpu_i32([0])
        out = ops.paged_attention(q, cache.k_cache, cache.v_cache, table, gpu_i32([0, 1]), gpu_i32([99, 59]), err_flag=flag)
        assert flag.item() == 1
        keep = [i for i in range(100) if i // 16 != 2]
        ref, _, tol, _ = attend_by_hand(q[0], cache.k[0][keep], cache.v[0][keep], len(keep) - 1, 1 / 8, 0)
        assert bool(((out[0].double().cpu() - ref).abs() <= tol).all())
        flag.zero_()
        ops.paged_attention(q, cache.k_cache, cache.v_cache, table, gpu_i32([0, 1]), gpu_i32([31, 59]), err_flag=flag)
        assert flag.item() == 0                                                        # a page that no row sees is not looked at
    flag = gpu_i32([0])
    out = torch.full_like(q, 2.0)
    ops.paged_attention(q, cache.k_cache, cache.v_cache, cache.table, gpu_i32([2, 10 ** 9]), gpu_i32([3, 3]), out=out, err_flag=flag)
    assert flag.item() == 1 and bool((out == 2.0).all())
    flag.zero_()
    ops.paged_attention(q, cache.k_cache, cache.v_cache, cache.table[:, :6], gpu_i32([0, 1]), gpu_i32([2 ** 31 - 1, 59]), err_flag=flag)
    assert flag.item() == 1


def test_attention_of_no_rows_and_no_pages(ops):
    cache = Cache(torch.float16, [30], 1, 32, 16, seed=14)
    empty = rows_q(cache, 0, 2, 32, torch.float16)
    none = gpu_i32([])
    assert ops.paged_attention(empty, cache.k_cache, cache.v_cache, cache.table, none, none).shape == (0, 2, 32)


def test_attention_far_pages(ops):
    """Offsets in the cache beyond 2^31 elements (and 2^32 bytes)."""
    dim, hk, page, pages = 256, 4, 64, 40000                                           # 2.6e9 elements of 2 bytes
    k_cache = torch.empty(pages, hk, page, dim, dtype=torch.bfloat16, device="cuda")
    v_cache = torch.empty_like(k_cache)
    ids = [39999, 1, 32769, 20000]
    gen = torch.Generator(device="cuda").manual_seed(15)
    k, v = (torch.randn(250, hk, dim, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    slot = torch.tensor([ids[i // page] * page + i % page for i in range(250)], device="cuda")
    position = torch.zeros(250, dtype=torch.int32, device="cuda")
    ops.rotary_store(None, k, v, k_cache, v_cache, position, slot, ops.rotary_frequencies(dim))
    q = torch.randn(1, 8, dim, generator=gen, device="cuda").to(torch.bfloat16)
    out = ops.paged_attention(q, k_cache, v_cache, gpu_i32([ids]), gpu_i32([0]), gpu_i32([249]))
    ref, _, tol, _ = attend_by_hand(q[0], k, v, 249, 1 / 16, 0)
    assert bool(((out[0].double().cpu() - ref).abs() <= tol).all())


def test_attention_of_single_pages_and_requests(ops):
    """The strides of dimensions of one element are of no consequence."""
    t = torch.float16
    cache = Cache(t, [11], 1, 64, 16, seed=23, spare=0)
    q = rows_q(cache, 1, 4, 64, t)
    ref, _, tol, _ = attend_by_hand(q[0], cache.k[0], cache.v[0], 10, 1 / 8, 0)
    shape = (1, 1, 16, 64)
    for stride in ((0, 1024, 64, 1), (1024, 5, 64, 1), (7, 0, 64, 1)):
        k, v = (c.as_strided(shape, stride) for c in (cache.k_cache, cache.v_cache))
        out = ops.paged_attention(q.as_strided((1, 4, 64), (3, 64, 1)), k, v, cache.table.t(), gpu_i32([0]), gpu_i32([10]))
        assert bool(((out[0].double().cpu() - ref).abs() <= tol).all()), stride


def test_attention_python_refusals(ops):
    cache = Cache(torch.bfloat16, [30], 2, 64, 16, seed=16)
    q = rows_q(cache, 2, 4, 64, torch.bfloat16)
    good = dict(q=q, k_cache=cache.k_cache, v_cache=cache.v_cache, table=cache.table, request=gpu_i32([0, 0]), position=gpu_i32([3, 4]))
    ops.paged_attention(**good)
    for bad in (dict(q=q.half()), dict(q=q[0]), dict(q=q[..., :32]), dict(q=rows_q(cache, 2, 3, 64, torch.bfloat16)), dict(q=q.cpu()),
                dict(table=cache.table.long()), dict(table=cache.table[0]), dict(request=gpu_i32([0])), dict(position=good["position"].long()),
                dict(out=q), dict(out=q.float()), dict(out=torch.zeros(2, 4, 32, dtype=torch.bfloat16, device="cuda")),
                dict(lse=torch.zeros(2, 3, device="cuda")), dict(lse=torch.zeros(2, 4, dtype=torch.float64, device="cuda")), dict(window=-1),
                dict(k_cache=cache.k_cache[:, :, :8], v_cache=cache.v_cache[:, :, :8])):
        with pytest.raises((ValueError, RuntimeError)):
            ops.paged_attention(**{**good, **bad})


# ---------------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("captured", [False, True])
def test_a_serving_loop(ops, dtype, captured):
    """Prompts come in, tokens follow, requests end and others take their place and their pages: every step's attention
    against the whole history in 64 bits.  Captured: the three calls as one graph, replayed every step with eager work and
    waits between, every replay checked."""
    t = TYPES[dtype]
    rng = random.Random(7)
    requests, width, page, hq, hk, dim, rows = 5, 12, 16, 4, 2, 64, 64
    pages = ops.new_pages(requests, width, 40)
    gen = torch.Generator(device="cuda").manual_seed(8)
    k_cache, v_cache = (torch.full((40, hk, page, dim), float("nan"), dtype=t, device="cuda") for _ in range(2))
    freq = ops.rotary_frequencies(dim, factor=2, scaling="linear")
    lengths, cursor, grow = pages.lengths.clone(), pages.cursor.clone(), torch.zeros(requests, dtype=torch.int32, device="cuda")
    qkv = torch.zeros(rows, hq + 2 * hk, dim, dtype=t, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    plan = ops.PagePlan(torch.empty(requests, **i32), torch.empty_like(cursor), torch.empty(requests + 1, **i32), torch.empty(rows, **i32),
                        torch.empty(rows, **i32), torch.empty(rows, dtype=torch.int64, device="cuda"), torch.empty(1, **i32))
    turned, out = torch.zeros(rows, hq, dim, dtype=t, device="cuda"), torch.zeros(rows, hq, dim, dtype=t, device="cuda")

    def step():
        ops.page_plan(lengths, grow, pages.table, pages.ring, cursor, page, out=plan)
        ops.rotary_store(qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:], k_cache, v_cache, plan.position, plan.slot, freq, out=turned)
        ops.paged_attention(turned, k_cache, v_cache, pages.table, plan.request, plan.position, out=out)

    graph = None
    if captured:
        step()                                     # nothing grows: no row, no page
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    held = [0] * requests
    keys, values = [[] for _ in held], [[] for _ in held]
    for n in range(25):
        g = []
        for s in range(requests):
            if held[s] == 0:
                g.append(rng.choice((0, rng.randint(1, 11))))
            else:
                g.append(-1 if rng.random() < 0.12 or held[s] > width * page - 12 else rng.choice((1, 1, 1, 3, 0)))
        grow.copy_(torch.tensor(g, dtype=torch.int32))
        qkv.copy_(torch.randn(rows, hq + 2 * hk, dim, generator=gen, device="cuda"))
        out.fill_(6.0)
        if graph:
            graph.replay()
        else:
            step()
        torch.cuda.synchronize()
        assert plan.status.item() == 0
        lengths.copy_(plan.lengths)
        cursor.copy_(plan.cursor)
        owned = [p for s in range(requests) for p in pages.table[s, :-(-int(lengths[s]) // page)].tolist()]
        free = [int(pages.ring[i % 40]) for i in range(*cursor.tolist())]
        assert sorted(owned + free) == list(range(40))              # every page has one owner
        row = 0
        for s in range(requests):
            if g[s] < 0:
                held[s], keys[s], values[s] = 0, [], []
                continue
            for _ in range(g[s]):
                at = torch.tensor([held[s]])
                keys[s].append(rotate_by_hand(qkv[row:row + 1, hq:hq + hk], at, freq, False, 1.0)[0].to(t)[0])
                values[s].append(qkv[row, hq + hk:].cpu())
                # the cache holds keys rounded after the rotation; where fp32 and 64 bits round to different neighbours the
                # key is a unit off, so the history takes what was stored once it has been found near
                stored = k_cache[int(plan.slot[row]) // page, :, int(plan.slot[row]) % page].cpu()
                unit = torch.finfo(t).eps
                assert bool(((stored.double() - keys[s][-1].double()).abs() <= unit * keys[s][-1].double().abs() + 2.0 ** -20).all())
                keys[s][-1] = stored
                assert int(plan.position[row]) == held[s]
                held[s] += 1
                ref, _, tol, _ = attend_by_hand(turned[row], torch.stack(keys[s]), torch.stack(values[s]), held[s] - 1, 1 / 8, 0)
                assert bool(((out[row].double().cpu() - ref).abs() <= tol).all()), (n, s, row)
                row += 1
        assert bool((out[row:] == 6.0).all())
        assert plan.start.tolist()[-1] == row


def test_calls_on_other_streams(ops):
    """The calls run on the current stream, and calls on two streams at once share nothing."""
    cache = Cache(torch.bfloat16, [4000, 2500], 2, 128, 16, seed=20)
    qs = [rows_q(cache, 2, 8, 128, torch.bfloat16) for _ in range(2)]
    request, position = gpu_i32([0, 1]), gpu_i32([3999, 2499])
    alone = [ops.paged_attention(q, cache.k_cache, cache.v_cache, cache.table, request, position) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_attention(qs[i], cache.k_cache, cache.v_cache, cache.table, request, position))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, alone[i])


def test_captured_calls_have_their_own_workspaces(ops):
    """Two graphs of calls that cut their work into pieces, replayed one after the other and side by side with eager calls between."""
    cache = Cache(torch.bfloat16, [9000, 700], 2, 64, 16, seed=24)
    request, position = gpu_i32([0, 1]), gpu_i32([8999, 699])
    qs = [rows_q(cache, 2, 8, 64, torch.bfloat16) for _ in range(3)]
    call = lambda q, out: ops.paged_attention(q, cache.k_cache, cache.v_cache, cache.table, request, position, out=out)      # noqa: E731
    alone = [call(q, torch.empty_like(q)) for q in qs]
    outs = [torch.empty_like(q) for q in qs]
    torch.cuda.synchronize()
    graphs = []
    for q, out in zip(qs[:2], outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(q, out)
            call(q, out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for n in range(8):
        for out in outs:
            out.fill_(n)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            if n % 2:
                with torch.cuda.stream(s):
                    g.replay()
            else:
                g.replay()
        call(qs[2], outs[2])
        torch.cuda.synchronize()
        for out, want in zip(outs, alone):
            assert torch.equal(out, want)


def test_the_same_call_gives_the_same_bytes(ops):
    cache = Cache(torch.float16, [3000, 1, 777], 2, 64, 16, seed=21)
    q = rows_q(cache, 3, 8, 64, torch.float16)
    call = lambda: ops.paged_attention(q, cache.k_cache, cache.v_cache, cache.table, gpu_i32([0, 1, 2]), gpu_i32([2999, 0, 776]))  # noqa: E731
    first = call()
    for _ in range(5):
        assert torch.equal(call(), first)
