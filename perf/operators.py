"""What the paged-cache operators are measured by: planning a step's pages and slots, rotating and storing its rows, and
attending from single rows over the cache.

`run` computes an operator in plain torch operations, or, where `own` is true, calls it as vits_amd offers it."""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one decoding step of a small serving batch: every request grows by one token
        dict(name="plan_step", op="plan", requests=48, page=16, context=2000, prompt=0, mix="step", pad=16, lens=1),
        # a step of a busy server: requests end, prompts come in, the rest decodes
        dict(name="plan_serving", op="plan", requests=700, page=32, context=4000, prompt=1500, mix="serving", pad=37, lens=2),
        # an offline job begins: nothing but prompts
        dict(name="plan_prompts", op="plan", requests=256, page=16, context=0, prompt=2000, mix="prompts", pad=0, lens=3),
        # one token of a model with this framework's encoder heads (2 heads of 96 channels, fp32)
        dict(name="rotary_one", op="rotary", rows=1, heads=2, kv_heads=2, dim=96, rotary=96, dtype="fp32", interleaved=False,
             page=16, context=700, scaling="none", prompt=False, pad=0),
        # a decoding batch far into long documents: half of each head turns, neighbours paired, frequencies interpolated
        dict(name="rotary_batch", op="rotary", rows=192, heads=32, kv_heads=8, dim=128, rotary=64, dtype="fp16", interleaved=True,
             page=16, context=500000, scaling="ramp", prompt=False, pad=11),
        # a prompt written to the cache in one go
        dict(name="rotary_prompt", op="rotary", rows=8192, heads=32, kv_heads=8, dim=128, rotary=128, dtype="bf16", interleaved=False,
             page=64, context=8192, scaling="base", prompt=True, pad=0),
        # one request, this framework's encoder heads, where latency is all that counts
        dict(name="attend_one", op="attend", requests=1, new=1, heads=2, kv_heads=2, dim=96, dtype="fp32", page=16, context=500, window=0,
             pad=0, lens=4),
        # the same heads in fp32, a batch of sentences
        dict(name="attend_sentences", op="attend", requests=100, new=1, heads=2, kv_heads=2, dim=96, dtype="fp32", page=16, context=2048,
             window=0, pad=4, lens=5),
        # an ordinary decoding batch with shared key-value heads and ragged lengths
        dict(name="attend_batch", op="attend", requests=64, new=1, heads=32, kv_heads=8, dim=128, dtype="bf16", page=16, context=4096,
             window=0, pad=0, lens=6),
        # one request over a very long context: there are few rows, so the length has to be split
        dict(name="attend_long", op="attend", requests=1, new=1, heads=32, kv_heads=8, dim=128, dtype="bf16", page=64, context=131072,
             window=0, pad=0, lens=7),
        # many short requests, every head with keys and values of its own
        dict(name="attend_many", op="attend", requests=512, new=1, heads=8, kv_heads=8, dim=64, dtype="fp16", page=32, context=1500,
             window=0, pad=0, lens=8),
        # drafted tokens are checked: up to five rows a request, a sliding window
        dict(name="attend_drafts", op="attend", requests=32, new=5, heads=16, kv_heads=2, dim=128, dtype="bf16", page=16, context=8000,
             window=1024, pad=3, lens=9),
    ]


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("plan", "rotary", "attend", "attend"))
    lens = rng.randrange(1 << 20)
    if op == "plan":
        mix = rng.choice(("step", "serving", "serving", "prompts"))
        requests, page = log_int(rng, 1, 4096), rng.choice((16, 32, 64, 128))
        context = 0 if mix == "prompts" else log_int(rng, 1, max(1, min(65536, 2000000 * page // requests)))
        prompt = 0 if mix == "step" else log_int(rng, 1, max(1, min(32768, 500000 // requests)))
        return dict(op=op, requests=requests, page=page, context=context, prompt=prompt, mix=mix, pad=rng.choice((0, rng.randrange(1, 200))), lens=lens)
    kv_heads, group, dim = rng.choice((1, 2, 4, 8)), rng.choice((1, 1, 2, 3, 4, 5, 8, 12, 16)), rng.choice((32, 64, 96, 128, 192, 256))
    dtype, page = rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.choice((16, 32, 48, 64, 128))
    if op == "rotary":
        rows = log_int(rng, 1, min(8192, 50000000 // ((group + 2) * kv_heads * dim)))
        prompt = rng.random() < 0.4
        return dict(op=op, rows=rows, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, rotary=rng.choice((dim, dim, dim // 2, dim // 4, dim - 10)),
                    dtype=dtype, interleaved=rng.random() < 0.5, page=page, context=max(rows, log_int(rng, 1, 1000000)),
                    scaling=rng.choice(("none", "linear", "base", "ramp")), prompt=prompt, pad=rng.choice((0, rng.randrange(0, rows))))
    requests = log_int(rng, 1, 512)
    new = rng.choice((1, 1, 1, rng.randrange(2, 9)))
    context = log_int(rng, 1, max(1, min(131072, 300000000 // (requests * (new + 1) * kv_heads * dim))))
    return dict(op=op, requests=requests, new=new, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, context=context,
                window=rng.choice((0, 0, 0, log_int(rng, 1, 4096))), pad=rng.choice((0, rng.randrange(0, 9))), lens=lens)


def lengths_of(case):
    """What a case's requests hold and how many tokens each gets, in an order that the seed changes afterwards. A growth of -1 ends a request."""
    rng, n = random.Random(case["lens"]), case["requests"]
    if case["op"] == "attend":
        held = [case["context"] if i == 0 else rng.randint(max(1, case["context"] // 16), case["context"]) for i in range(n)]
        return held, [min(h, rng.randint(1, case["new"])) for h in held]
    held, grow = [], []
    for _ in range(n):
        what = {"step": 1.0, "prompts": 0.0}.get(case["mix"], rng.random())
        cached, prompt = (rng.randint(1, case["context"]) if case["context"] else 0), (rng.randint(1, case["prompt"]) if case["prompt"] else 0)
        # of a serving step's requests an eighth begins, an eighth ends, a sixteenth waits and the rest gets one token
        h, g = (0, prompt) if what < 0.125 else (cached, -1) if what < 0.25 else (cached, 0) if what < 0.3125 else (cached, 1)
        held.append(h)
        grow.append(g)
    return held, grow


def pages_for(tokens, page):
    return -(-tokens // page)


def shuffled_table(held, page, width, pages, gen):
    """A block table whose requests hold pages spread over the pool, and the pages that nobody holds."""
    order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32)
    count = (held + page - 1) // page
    table = torch.full((held.numel(), width), -1, dtype=torch.int32, device="cuda")
    mine = torch.arange(width, device="cuda")[None, :] < count[:, None]
    taken = int(count.sum())
    table[mine] = order[:taken]
    return table, order[taken:]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"plan": prepare_plan, "rotary": prepare_rotary, "attend": prepare_attend}[case["op"]](case, gen)


def prepare_plan(case, gen):
    held, grow = (torch.tensor(x, device="cuda") for x in lengths_of(case))
    order = torch.randperm(case["requests"], generator=gen, device="cuda")
    held, grow = held[order], grow[order]
    page, after = case["page"], held + grow.clamp(min=0)
    width = pages_for(int(after.max()), page) + 1
    need = int(((after + page - 1) // page).sum())
    pages = need + need // 8 + 16
    table, free = shuffled_table(held, page, width, pages, gen)
    # the free pages lie in a ring that has been round some times
    head = pages * 5 + int(torch.randint(0, pages, (1,), generator=gen, device="cuda"))
    ring = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    ring[(head + torch.arange(free.numel(), device="cuda")) % pages] = free
    n, rows = case["requests"], int(grow.clamp(min=0).sum()) + case["pad"]
    i32 = dict(dtype=torch.int32, device="cuda")
    out = (torch.empty(n, **i32), torch.empty(2, dtype=torch.int64, device="cuda"), torch.empty(n + 1, **i32), torch.empty(rows, **i32),
           torch.empty(rows, **i32), torch.empty(rows, dtype=torch.int64, device="cuda"), torch.empty(1, **i32))
    return dict(op="plan", lengths=held.to(torch.int32), grow=grow.to(torch.int32), table=table, ring=ring, page=page, rows=rows, out=out,
                cursor=torch.tensor([head, head + free.numel()], dtype=torch.int64, device="cuda"))


def frequencies(case):
    """Radians a position for each pair: base^(-2i / n), as it is or stretched fourfold for long contexts in one of three ways."""
    n = case["rotary"]
    i = torch.arange(0, n, 2, dtype=torch.float64)
    base = 10000.0 * (4.0 ** (n / max(1, n - 2)) if case["scaling"] == "base" else 1.0)
    freq = base ** (-i / n)
    if case["scaling"] == "linear":
        freq = freq / 4
    if case["scaling"] == "ramp":  # slow pairs are interpolated, fast ones kept, those between are blended
        turns = 4096 * freq / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        freq = freq / 4 * (1 - keep) + freq * keep
    return freq.cuda()


def prepare_rotary(case, gen):
    rows, hq, hk, d, page = case["rows"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    dtype = DTYPES[case["dtype"]]
    qkv = torch.randn(rows, hq + 2 * hk, d, generator=gen, device="cuda").to(dtype)
    pages = pages_for(rows, page) + 8
    k_cache, v_cache = (torch.randn(pages, hk, page, d, generator=gen, device="cuda").to(dtype) for _ in range(2))
    if case["prompt"]:  # one request's rows: consecutive positions, consecutive slots of shuffled pages
        first = int(torch.randint(0, case["context"] - rows + 1, (1,), generator=gen, device="cuda"))
        at = torch.arange(rows, device="cuda")
        position, order = first + at, torch.randperm(pages, generator=gen, device="cuda")
        slot = order[at // page] * page + at % page
    else:
        position = torch.randint(0, case["context"], (rows,), generator=gen, device="cuda")
        slot = torch.randperm(pages * page, generator=gen, device="cuda")[:rows]
    slot[rows - case["pad"]:] = -1
    return dict(op="rotary", q=qkv[:, :hq], k=qkv[:, hq:hq + hk], v=qkv[:, hq + hk:], k_cache=k_cache, v_cache=v_cache, slot=slot,
                position=position.to(torch.int32), freq=frequencies(case), scale=1.1386 if case["scaling"] == "ramp" else 1.0,
                interleaved=case["interleaved"], out=torch.zeros(rows, hq, d, dtype=dtype, device="cuda"))


def prepare_attend(case, gen):
    held, new = (torch.tensor(x, device="cuda") for x in lengths_of(case))
    order = torch.randperm(case["requests"], generator=gen, device="cuda")
    held, new = held[order], new[order]
    page, hk, d, dtype = case["page"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    width = pages_for(case["context"], page)
    need = int(((held + page - 1) // page).sum())
    pages = need + need // 16 + 1
    table, _ = shuffled_table(held, page, width, pages, gen)
    k_cache, v_cache = (torch.randn(pages, hk, page, d, generator=gen, device="cuda", dtype=dtype) for _ in range(2))
    rows, total = int(new.sum()) + case["pad"], int(new.sum())
    request = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    position = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    request[:total] = torch.repeat_interleave(torch.arange(case["requests"], device="cuda"), new).to(torch.int32)
    first = torch.cumsum(new, 0) - new
    mine = request[:total].long()
    position[:total] = (held[mine] - new[mine] + torch.arange(total, device="cuda") - first[mine]).to(torch.int32)
    q = torch.randn(rows, case["heads"], d, generator=gen, device="cuda").mul_(1.5).to(dtype)
    return dict(op="attend", q=q, k_cache=k_cache, v_cache=v_cache, table=table, request=request, position=position, window=case["window"],
                scale=1 / math.sqrt(d), max_keys=case["context"], out=torch.zeros_like(q),
                lse=torch.zeros(rows, case["heads"], dtype=torch.float32, device="cuda"))


def run(s):
    if own:
        from vits_amd import ops
        if s["op"] == "plan":
            ops.page_plan(s["lengths"], s["grow"], s["table"], s["ring"], s["cursor"], s["page"], out=s["out"])
            return [s["table"], s["ring"], *s["out"]]
        if s["op"] == "rotary":
            ops.rotary_store(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["position"], s["slot"], s["freq"], interleaved=s["interleaved"],
                             scale=s["scale"], out=s["out"])
            return [s["out"], s["k_cache"], s["v_cache"]]
        ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["request"], s["position"], scale=s["scale"], window=s["window"],
                            max_keys=s["max_keys"], out=s["out"], lse=s["lse"])
        return [s["out"], s["lse"]]
    return {"plan": plain_plan, "rotary": plain_rotary, "attend": plain_attend}[s["op"]](s)


def plain_plan(s):
    lengths, grow, page, table, ring = s["lengths"].long(), s["grow"].long(), s["page"], s["table"], s["ring"]
    head, tail = s["cursor"][0], s["cursor"][1]
    add, ends = grow.clamp(min=0), grow < 0
    held = (lengths + page - 1) // page
    fresh = (lengths + add + page - 1) // page - held
    back = torch.where(ends, held, torch.zeros_like(held))
    row_end, fresh_end, back_end = add.cumsum(0), fresh.cumsum(0), back.cumsum(0)
    row = torch.arange(s["rows"], device="cuda")
    mine = torch.searchsorted(row_end, row, right=True)
    live = mine < lengths.numel()
    request = mine.clamp(max=lengths.numel() - 1)
    position = lengths[request] + row - (row_end - add)[request]
    # a request's first new row of a page takes the next free page
    nth = position // page - held[request]
    taken = ring[(head + (fresh_end - fresh)[request] + nth.clamp(min=0)) % ring.numel()]
    new_page = live & (nth >= 0)
    opens = new_page & ((position % page == 0) | (row == (row_end - add)[request]))
    table[request[opens], (position // page)[opens]] = taken[opens]
    page_of = torch.where(new_page, taken, table[request, (position // page).clamp(max=table.shape[1] - 1)]).long()
    # pages of requests that end go to the ring's other end
    at = torch.arange(table.shape[1], device="cuda")[None, :]
    gone = at < back[:, None]
    ring[((tail + (back_end - back)[:, None] + at) % ring.numel())[gone]] = table[gone]
    none = torch.full_like(row, -1)
    lengths_out, cursor, start, request_out, position_out, slot, status = s["out"]
    lengths_out.copy_(torch.where(ends, torch.zeros_like(lengths), lengths + add))
    cursor.copy_(torch.stack((head + fresh_end[-1], tail + back_end[-1])))
    start.copy_(torch.cat((torch.zeros_like(row_end[:1]), row_end)))
    request_out.copy_(torch.where(live, request, none))
    position_out.copy_(torch.where(live, position, none))
    slot.copy_(torch.where(live, page_of * page + position % page, none))
    status.zero_()
    return [table, ring, *s["out"]]


def turned(x, cos, sin, interleaved):
    n = 2 * cos.shape[-1]
    x = x.float()
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., :n // 2], x[..., n // 2:n])
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.cat((torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1), x[..., n:]), -1)


def plain_rotary(s):
    angle = s["position"].double()[:, None] * s["freq"]
    cos, sin = ((f(angle) * s["scale"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    live, dtype, page = s["slot"] >= 0, s["q"].dtype, s["k_cache"].shape[2]
    s["out"].copy_(torch.where(live[:, None, None], turned(s["q"], cos, sin, s["interleaved"]).to(dtype), s["out"]))
    slot = s["slot"][live]
    s["k_cache"][slot // page, :, slot % page] = turned(s["k"], cos, sin, s["interleaved"]).to(dtype)[live]
    s["v_cache"][slot // page, :, slot % page] = s["v"][live]
    return [s["out"], s["k_cache"], s["v_cache"]]


def plain_attend(s):
    q, table, position = s["q"], s["table"], s["position"].long()
    rows, heads, d = q.shape
    pages, kv_heads, page, _ = s["k_cache"].shape
    mine = table[s["request"].clamp(min=0).long()].clamp(min=0).long()
    k, v = (c[mine].permute(0, 2, 1, 3, 4).reshape(rows, kv_heads, -1, d).float() for c in (s["k_cache"], s["v_cache"]))
    at = torch.arange(k.shape[2], device="cuda")[None, :]
    seen = at <= position[:, None]
    if s["window"]:
        seen &= at > position[:, None] - s["window"]
    seen = seen[:, None, None, :]
    score = torch.matmul(q.float().view(rows, kv_heads, heads // kv_heads, d), k.transpose(-1, -2)) * s["scale"]
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    o = torch.matmul(weight, torch.where(seen.transpose(-1, -2), v, torch.zeros_like(v))) / total
    o = torch.where(total > 0, o, torch.zeros_like(o)).view(rows, heads, d)
    lse = (top + total.log()).view(rows, heads)
    live = (s["request"] >= 0)[:, None]
    s["out"].copy_(torch.where(live[..., None], o.to(q.dtype), s["out"]))
    s["lse"].copy_(torch.where(live, lse, s["lse"]))
    return [s["out"], s["lse"]]


def work(case):
    held, grow = lengths_of(case) if case["op"] != "rotary" else (None, None)
    if case["op"] == "plan":
        page = case["page"]
        add = [max(g, 0) for g in grow]
        fresh = sum(pages_for(h + a, page) - pages_for(h, page) for h, a in zip(held, add))
        back = sum(pages_for(h, page) for h, g in zip(held, grow) if g < 0)
        rows = sum(add) + case["pad"]
        # lengths and growths in, lengths and row starts out, pages in and out, 16 bytes a row
        return {"bytes": 16 * len(held) + 8 * (fresh + back) + 16 * rows + 40, "flops": 8 * (len(held) + rows)}
    size = 4 if case["dtype"] == "fp32" else 2
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        rows = case["rows"] - case["pad"]
        return {"bytes": rows * 2 * (hq + 2 * hk) * d * size + 12 * case["rows"] + 4 * case["rotary"], "flops": rows * (hq + hk) * case["rotary"] * 3}
    seen = keys = rows = 0
    for h, n in zip(held, grow):
        lows = [max(0, h - n + i + 1 - case["window"]) if case["window"] else 0 for i in range(n)]
        seen += sum(h - n + i + 1 - low for i, low in enumerate(lows))
        keys += h - lows[0]
        rows += n
    return {"bytes": 2 * keys * hk * d * size + rows * hq * (2 * d * size + 4) + 4 * sum(pages_for(h, case["page"]) for h in held) + 8 * rows,
            "flops": 4 * seen * hq * d}


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    return exact_rotary(s) if case["op"] == "rotary" else exact_attend(s)


def exact_rotary(s):
    pairs = s["freq"].numel()
    angle = s["position"].to(torch.float64).view(-1, 1, 1) * s["freq"].view(1, 1, -1)
    spin = torch.polar(torch.full_like(angle, s["scale"]), angle)
    live = (s["slot"] >= 0).nonzero()[:, 0]

    def turn(x):
        x = x.to(torch.float64).clone()
        lead = x[..., :2 * pairs]
        z = torch.complex(lead[..., 0::2], lead[..., 1::2]) if s["interleaved"] else torch.complex(lead[..., :pairs], lead[..., pairs:])
        z = z * spin
        if s["interleaved"]:
            x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2] = z.real, z.imag
        else:
            x[..., :pairs], x[..., pairs:2 * pairs] = z.real, z.imag
        return x

    out, k_cache, v_cache = (s[n].to(torch.float64) for n in ("out", "k_cache", "v_cache"))
    page = k_cache.shape[2]
    slots, offsets = s["slot"][live] // page, s["slot"][live] % page
    out[live] = turn(s["q"])[live]
    k_cache.transpose(1, 2)[slots, offsets] = turn(s["k"])[live]
    v_cache.transpose(1, 2)[slots, offsets] = s["v"].to(torch.float64)[live]
    return [out, k_cache, v_cache]


def exact_attend(s):
    out, lse = s["out"].to(torch.float64), s["lse"].to(torch.float64)
    kv_heads, page, d = s["k_cache"].shape[1:]
    group = s["q"].shape[1] // kv_heads
    for row, (request, position) in enumerate(zip(s["request"].tolist(), s["position"].tolist())):
        if request < 0:
            continue
        low = max(0, position + 1 - s["window"]) if s["window"] else 0
        at = torch.arange(low, position + 1, device="cuda")
        where = s["table"][request].long()[at // page]
        k, v = (c[where, :, at % page].to(torch.float64).transpose(0, 1).contiguous() for c in (s["k_cache"], s["v_cache"]))  # [kv_heads, keys, d]
        score = torch.bmm(k, s["q"][row].to(torch.float64).view(kv_heads, group, d).transpose(1, 2).contiguous()) * s["scale"]
        lse[row] = torch.logsumexp(score, 1).view(-1)
        weight = torch.softmax(score, 1).transpose(1, 2).contiguous()
        out[row] = torch.bmm(weight, v).reshape(-1, d)
    return [out, lse]
