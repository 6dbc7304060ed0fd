"""The operators for a step of several sequences, as cases that can be timed.

The user is an engine that serves more than one conversation at a time. Each step it hands the
backend a batch: sequence s has ``start`` positions in a paged Q8_0 cache and ``new`` tokens of
its own; the new rows of all sequences lie one behind the other. Kinds of case:

  store   quantise the new keys and values into the sequences' pages, and hand back what the
          cache now stands for
  load    read whole sequences back from the pages
  paged   causal grouped attention of the new tokens over the paged cache (their own keys are
          already in it): single tokens, drafted runs, prompt chunks, and mixtures
  packed  causal grouped attention of whole prompts of different lengths, keys and values in hand
  verify  drafted tokens against the target's probabilities, from given random numbers

Head layouts are those of the models in ``sulimo_amd.synthetic`` and the tests' small one.
"""
import math
import random

import numpy as np
import torch

own = False

HEADS = {"1.5b": (12, 2, 128), "3b": (24, 8, 128), "small": (4, 2, 64)}  # query heads, key heads, head size


def _case(**c):
    """A case of plain values: a range (lo, hi) becomes two of them."""
    out = {}
    for k, v in c.items():
        if isinstance(v, list):
            out[k + "_lo"], out[k + "_hi"] = v
        else:
            out[k] = v
    return out


def listed():
    return [
        # one decoding step of 16 conversations: the smallest call, launch and latency count
        _case(name="store_step_16", kind="store", heads="1.5b", seqs=16, new=[1, 1], start=[100, 4000], page=64, shape=1),
        # prompts of several users at once, ragged lengths
        _case(name="store_prompts", kind="store", heads="3b", seqs=7, new=[150, 4000], start=[0, 500], page=64, shape=2),
        # a conversation's cache read back, a page size that is no power of two
        _case(name="load_turn", kind="load", heads="1.5b", seqs=1, new=[23, 23], start=[777, 777], page=48, shape=3),
        # many long conversations read back
        _case(name="load_many", kind="load", heads="3b", seqs=12, new=[1, 1], start=[2000, 8000], page=128, shape=4),
        # one conversation decoding
        _case(name="decode_1", kind="paged", heads="1.5b", seqs=1, new=[1, 1], start=[2047, 2047], page=16, window=0, shape=5),
        # a full server decoding: the largest cache
        _case(name="decode_64", kind="paged", heads="3b", seqs=64, new=[1, 1], start=[500, 8000], page=64, window=0, shape=6),
        # four drafted tokens behind the last one of 16 conversations
        _case(name="drafts_16", kind="paged", heads="1.5b", seqs=16, new=[5, 5], start=[200, 4000], page=32, window=0, shape=7),
        # chunks of two long prompts beside 30 decoding conversations
        _case(name="chunks_mixed", kind="paged", heads="3b", seqs=32, chunks=2, new=[400, 700], start=[300, 7000], page=64, window=0,
             shape=8),
        # a few short prompts of a small model
        _case(name="packed_small", kind="packed", heads="small", seqs=5, new=[1, 130], window=0, shape=9),
        # whole prompts of several users: the most products
        _case(name="packed_prompts", kind="packed", heads="3b", seqs=8, new=[500, 4096], window=0, shape=10),
        # four drafts of one conversation, full vocabulary
        _case(name="verify_1", kind="verify", vocab=151936, seqs=1, new=[5, 5], point=False, temp=0.8, shape=11),
        # up to eight drafts of 24 conversations
        _case(name="verify_24", kind="verify", vocab=151936, seqs=24, new=[1, 9], point=False, temp=1.0, shape=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _range(rng, lo, hi):
    a, b = _log_int(rng, lo, hi), _log_int(rng, lo, hi)
    return [min(a, b), max(a, b)]


def draw(rng):
    kind = rng.choice(["store", "load", "paged", "paged", "paged", "packed", "packed", "verify"])
    c = dict(kind=kind, shape=rng.randrange(1 << 30))
    if kind == "verify":
        c.update(vocab=rng.choice([151936, 128256, 32000, _log_int(rng, 100, 150000)]), seqs=_log_int(rng, 1, 24), new=_range(rng, 1, 9),
                 point=rng.random() < 0.3, temp=rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.5]))
        return _case(**c)
    c["heads"] = rng.choice(sorted(HEADS))
    page = rng.choice([8, 16, 16, 32, 48, 64, 64, 100, 128, 256])
    window = rng.choice([0, 0, 0, rng.randrange(1, 3000)])
    if kind == "store":
        new = _range(rng, 1, 4000)
        c.update(seqs=_log_int(rng, 1, max(1, min(64, 25000 // new[1]))), new=new, start=_range(rng, 1, 4000), page=page)
    elif kind == "load":
        start = _range(rng, 1, 8000)
        c.update(seqs=_log_int(rng, 1, max(1, min(64, 90000 // start[1]))), new=[0, 1], start=start, page=page)
    elif kind == "packed":
        new = _range(rng, 1, 4096)
        c.update(seqs=_log_int(rng, 1, max(1, min(32, 4096 * 3 // new[1]))), new=new, window=window)
    else:
        form = rng.choice(["decode", "drafts", "chunk", "mixed"])
        start = _range(rng, 1, 8000)
        if form == "decode":
            c.update(seqs=_log_int(rng, 1, min(64, 270000 // start[1])), new=[1, 1], start=start)
        elif form == "drafts":
            c.update(seqs=_log_int(rng, 1, 32), new=_range(rng, 2, 24), start=start)
        elif form == "chunk":
            c.update(seqs=rng.choice([1, 1, 2]), new=_range(rng, 10, 1024), start=start)
        else:
            c.update(seqs=_log_int(rng, 2, 40), chunks=1, new=_range(rng, 10, 1024), start=start)
        c.update(page=page, window=window)
    return _case(**c)


def _lens(case):
    """(positions in the cache, new tokens) of each sequence: a function of the case alone."""
    r = random.Random(case["shape"])
    start, new = [], []
    for s in range(case["seqs"]):
        chunk = s >= case["seqs"] - case.get("chunks", case["seqs"])  # the long ones come last
        new.append(r.randint(case["new_lo"], case["new_hi"]) if chunk else 1)
        start.append(r.randint(case["start_lo"], case["start_hi"]) if "start_lo" in case else 0)
    return start, new


# ---- inputs ----

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)


def _pages(case, seed):
    """(page_table uint32 [seqs][most], pages): the sequences' pages in mixed order, a tenth more than used."""
    start, new = _lens(case)
    need = [-(-(a + b) // case["page"]) for a, b in zip(start, new)]
    pages = sum(need) + max(1, sum(need) // 10)
    order = np.random.RandomState(int(seed) & 0x7FFFFFFF).permutation(pages).astype(np.uint32)
    table = np.zeros((len(need), max(1, max(need))), np.uint32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, pages


def _cache(g, pages, page, width):
    """A Q8_0 cache as attention meets it: N(0, 1) values in blocks of 32, uint8 [pages * page, width / 32, 34]."""
    rows = pages * page
    out = torch.empty((rows, width // 32, 34), dtype=torch.uint8, device="cuda")
    for r in range(0, rows, 65536):
        v = torch.randn((min(65536, rows - r), width // 32, 32), generator=g, device="cuda")
        d = v.abs().amax(-1, keepdim=True) / 127.0
        out[r:r + 65536, :, :2] = d.half().view(torch.uint8)
        out[r:r + 65536, :, 2:] = torch.round(v / d).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return out


def _inputs(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    start, new = _lens(case)
    T = sum(new)
    if kind == "verify":
        # the draft model's distribution is the target's with noise; the drafts are drawn from it
        V = case["vocab"]
        logits = 2.0 * torch.randn((T, V), generator=g, device="cuda")
        near = (logits[:-1] + 0.7 * torch.randn((T - 1, V), generator=g, device="cuda")) if T > 1 else logits[:0]
        probs = torch.softmax(near, -1)
        tokens = torch.randint(0, V, (T,), generator=g, device="cuda", dtype=torch.int32)
        off = 0
        rows = []  # logits row that a drafted token is judged by
        for n in new:
            rows += range(off, off + n - 1)
            off += n
        rows = torch.tensor(rows, dtype=torch.long, device="cuda")
        probs = probs[rows].contiguous()
        if rows.numel():
            tokens[rows + 1] = (probs.argmax(-1) if case["point"] else torch.multinomial(probs, 1, generator=g)[:, 0]).int()
        return dict(logits=logits, tokens=tokens, probs=None if case["point"] else probs,
                    u=torch.rand((T,), generator=g, device="cuda"))
    H, Hk, hd = HEADS[case["heads"]]
    i = {}
    if kind in ("paged", "packed"):
        i["q"] = torch.randn((T, H, hd), generator=g, device="cuda").half()
    if kind in ("store", "packed"):
        for n in ("k", "v"):
            i[n] = torch.randn((T, Hk, hd), generator=g, device="cuda").half()
    if kind != "packed":
        i["table"], i["pages"] = _pages(case, seed)
        if kind != "store":
            for n in ("k_cache", "v_cache"):
                i[n] = _cache(g, i["pages"], case["page"], Hk * hd)
    return i


class _Memory:
    """A library buffer as torch sees device memory; it keeps the buffer alive."""

    def __init__(self, buf, shape, typestr):
        from sulimo_amd import hip
        self.buf = buf
        ptr = hip.lib().sulimo_hip_buffer_device_ptr(buf.handle)
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (int(ptr), False), "version": 3}


_TYPES = {torch.float16: "<f2", torch.float32: "<f4", torch.uint8: "|u1", torch.int32: "<i4"}


def _buf(ctx, shape, dtype, fill=None):
    """(a library buffer, torch's view of it)."""
    from sulimo_amd import hip
    n = max(1, math.prod(shape)) * torch.empty((), dtype=dtype).element_size()
    b = hip.HipBuffer.device_only(ctx, n)
    v = torch.as_tensor(_Memory(b, shape, _TYPES[dtype]), device="cuda") if math.prod(shape) else torch.empty(shape, dtype=dtype, device="cuda")
    if fill is not None:
        v.copy_(fill)
    return b, v


def prepare(case, seed):
    i = _inputs(case, seed)
    start, new = _lens(case)
    st = dict(case=case, start=start, new=new)
    if not own:
        st.update(i)
        if case["kind"] == "store":
            H, Hk, hd = HEADS[case["heads"]]
            for n in ("k_cache", "v_cache"):
                st[n] = torch.zeros((i["pages"] * case["page"], Hk * hd // 32, 34), dtype=torch.uint8, device="cuda")
        if case["kind"] == "verify":
            off = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
            st["off"], st["count"] = torch.tensor(off[:-1], device="cuda"), torch.tensor(new, device="cuda")
        else:
            if "table" in i:
                st["slots"] = _slots(case, i["table"], start, new)
        torch.cuda.synchronize()
        return st
    from sulimo_amd import hip
    ctx = hip.HipContext.get_or_init(0)
    T, kind = sum(new), case["kind"]
    st["ctx"] = ctx
    for n, t in i.items():
        if isinstance(t, torch.Tensor):
            st[n] = _buf(ctx, t.shape, t.dtype, t)[0]
    if kind == "verify":
        batch = hip.SeqBatch(ctx)
        batch.set(new)
        st["probs"] = st.get("probs")
        st["accepted"], accepted = _buf(ctx, (len(new),), torch.int32)
        st["answer"], answer = _buf(ctx, (T,), torch.int32)
        st["out"] = dict(accepted=accepted, answer=answer)
    else:
        H, Hk, hd = HEADS[case["heads"]]
        batch = hip.SeqBatch(ctx, H, Hk, hd, window=case.get("window", 0), page_size=case.get("page", 0), n_pages=i.get("pages", 0))
        batch.set(new, start, i.get("table"))
        if kind == "store":
            scales = {}
            for n in ("k_cache", "v_cache"):
                shape = (i["pages"] * case["page"], Hk * hd // 32, 34)
                st[n], cache = _buf(ctx, shape, torch.uint8, torch.zeros(shape, dtype=torch.uint8, device="cuda"))
                scales[n + "_scales"] = _scales(cache)
        if kind in ("store", "load"):
            rows = T if kind == "store" else T + sum(start)
            st["k_out"], k = _buf(ctx, (rows, Hk * hd), torch.float16)
            st["v_out"], v = _buf(ctx, (rows, Hk * hd), torch.float16)
            st["out"] = dict(k=k, v=v, **(scales if kind == "store" else {}))
        else:
            st["y"], st["out"] = _buf(ctx, (T, H, hd), torch.float16)
    st["batch"] = batch
    torch.cuda.synchronize()
    return st


def _scales(cache):
    """The scales of a cache's blocks, a view of it."""
    return cache.view(torch.float16)[..., 0]


def _slots(case, table, start, new):
    """Cache rows of each sequence's positions 0 .. start + new - 1, one tensor a sequence."""
    P, out = case["page"], []
    for s, (a, n) in enumerate(zip(start, new)):
        p = np.arange(a + n)
        out.append(torch.from_numpy(table[s][p // P].astype(np.int64) * P + p % P).cuda())
    return out


# ---- one pass ----

def run(st):
    if own:
        return _run_own(st)
    kind = st["case"]["kind"]
    if kind == "store":
        return _plain_store(st)
    if kind == "load":
        return dict(k=_plain_rows(st["k_cache"], torch.cat(st["slots"])).half(), v=_plain_rows(st["v_cache"], torch.cat(st["slots"])).half())
    if kind == "verify":
        return _plain_verify(st)
    return _plain_attention(st)


def _run_own(st):
    from sulimo_amd import hip
    c, ctx, batch, kind = st["case"], st["ctx"], st["batch"], st["case"]["kind"]
    if kind == "store":
        hip.enqueue_kv_store_paged(ctx, batch, st["k"], st["v"], st["k_cache"], st["v_cache"], st["k_out"], st["v_out"])
    elif kind == "load":
        hip.enqueue_kv_load_paged(ctx, batch, st["k_cache"], st["v_cache"], st["k_out"], st["v_out"])
    elif kind == "paged":
        hip.enqueue_attention_paged(ctx, batch, st["q"], st["k_cache"], st["v_cache"], st["y"])
    elif kind == "packed":
        hip.enqueue_attention_packed(ctx, batch, st["q"], st["k"], st["v"], st["y"])
    else:
        hip.enqueue_verify_drafts(ctx, batch, st["logits"], st["tokens"], st["probs"], st["u"], c["vocab"], c["temp"],
                                  st["accepted"], st["answer"])
    return st["out"]


def _plain_store(st):
    """d = max|x| / 127, code = round half away(x * (1 / d)) in 32 bits, as the ring's format lays down."""
    new, out = st["new"], {}
    at = torch.cat([s[len(s) - n:] for s, n in zip(st["slots"], new)])
    for name in ("k", "v"):
        x = st[name].float()
        b = x.reshape(x.shape[0], -1, 32)
        d = b.abs().amax(-1, keepdim=True) / 127.0
        y = b * torch.where(d != 0, 1.0 / d, 0.0)
        t = torch.trunc(y)
        code = (t + torch.where((y - t).abs() >= 0.5, torch.sign(y), 0.0)).clamp(-128, 127)
        blocks = torch.cat([d.half().view(torch.uint8), code.to(torch.int8).view(torch.uint8)], -1)
        st[name + "_cache"][at] = blocks
        out[name] = (code * d.half().float()).half().flatten(1)
        out[name + "_cache_scales"] = _scales(st[name + "_cache"])
    return out


def _plain_rows(cache, slots):
    """f32 [rows, width]: code * scale of the cache rows."""
    b = cache[slots]
    d = b[..., :2].contiguous().view(torch.float16).float()
    return (b[..., 2:].contiguous().view(torch.int8).float() * d).flatten(1)


def _plain_attention(st):
    c = st["case"]
    H, Hk, hd = HEADS[c["heads"]]
    G, w, out, off = H // Hk, c["window"], [], 0
    for s, (a, n) in enumerate(zip(st["start"], st["new"])):
        if n == 0:
            continue
        q = st["q"][off:off + n].float()
        if c["kind"] == "paged":
            k, v = (_plain_rows(st[x], st["slots"][s]).reshape(a + n, Hk, hd) for x in ("k_cache", "v_cache"))
        else:
            k, v = st["k"][off:off + n].float(), st["v"][off:off + n].float()
        k, v = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()  # [Hk, hd, keys], [Hk, keys, hd]
        p = torch.arange(a + n, device="cuda")
        for t in range(0, n, 1024):
            m = min(1024, n - t)
            qt = q[t:t + m].reshape(m, Hk, G, hd).permute(1, 2, 0, 3).reshape(Hk, G * m, hd)
            x = (torch.matmul(qt, k) / math.sqrt(hd)).reshape(Hk, G, m, a + n)
            at = a + t + torch.arange(m, device="cuda")[:, None]
            hide = (p > at) | (p <= at - w) if w else p > at
            x = torch.where(hide, -math.inf, x)
            e = torch.exp(x - x.amax(-1, keepdim=True))
            y = torch.matmul(e.reshape(Hk, G * m, a + n), v) / e.sum(-1).reshape(Hk, G * m, 1)
            out.append(y.reshape(Hk, G, m, hd).permute(2, 0, 1, 3).reshape(m, H, hd).half())
        off += n
    return torch.cat(out) if out else st["q"]


def _argmax(x):
    """The greatest entry's index, the last one where several are (as the framework's top-1)."""
    return x.shape[-1] - 1 - x.flip(-1).argmax(-1)


def _plain_verify(st):
    """In 64 bits throughout: a running sum over the vocabulary next to a border."""
    c, logits, off, count = st["case"], st["logits"], st["off"], st["count"]
    V, S, most = c["vocab"], len(st["new"]), max(st["new"])
    T = logits.shape[0]
    k = count - 1  # drafts of each sequence
    i = torch.arange(most, device="cuda")
    row = (off[:, None] + i).clamp(max=T - 1)                    # [S, most] the row that judges draft i
    drafted = i < k[:, None]
    d = st["tokens"].long()[(row + 1).clamp(max=T - 1)]
    prow = (off - torch.arange(S, device="cuda"))[:, None] + i   # its row of the draft's probabilities
    if c["temp"] == 0:
        top = _argmax(logits)
        ok = drafted & (top[row] == d)
    else:
        x = logits.double() / c["temp"]
        e = torch.exp(x - x.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
        q = 1.0 if st["probs"] is None else st["probs"].double()[prow.clamp(max=st["probs"].shape[0] - 1), d] if st["probs"].shape[0] else 1.0
        ok = drafted & (st["u"].double()[row] * q < p[row, d])
    a = ok.long().cumprod(-1).sum(-1)                            # accepted drafts
    last = off + a
    if c["temp"] == 0:
        tok = top[last]
    else:
        w = p[last]
        rejected = a < k
        ar = a.clamp(max=most - 1)[:, None]
        if st["probs"] is None:
            r = torch.where(torch.arange(V, device="cuda") == d.gather(1, ar), 0.0, w)
        elif st["probs"].shape[0]:
            r = (w - st["probs"].double()[prow.gather(1, ar)[:, 0].clamp(max=st["probs"].shape[0] - 1)]).clamp(min=0.0)
        else:
            r = w
        w = torch.where((rejected & (r.sum(-1) > 0))[:, None], r, w)
        cum = w.cumsum(-1)
        tok = (cum <= st["u"].double()[off + k][:, None] * cum[:, -1:]).sum(-1)
        tok = torch.minimum(tok, _argmax((w > 0).int()))
    seq = torch.repeat_interleave(torch.arange(S, device="cuda"), count, output_size=T)
    j = torch.arange(T, device="cuda") - off[seq]
    nxt = st["tokens"].long()[(torch.arange(T, device="cuda") + 1).clamp(max=T - 1)]
    answer = torch.where(j < a[seq], nxt, torch.where(j == a[seq], tok[seq], -1))
    return dict(accepted=a.int(), answer=answer.int())


# ---- what a pass cannot do without ----

def work(case):
    start, new = _lens(case)
    T, kind = sum(new), case["kind"]
    if kind == "verify":
        rows = T + (0 if case["point"] or case["temp"] == 0 else case["seqs"])
        return dict(bytes=4.0 * case["vocab"] * rows + 12.0 * T, flops=4.0 * case["vocab"] * T)
    H, Hk, hd = HEADS[case["heads"]]
    width = Hk * hd
    if kind == "store":
        return dict(bytes=2 * T * width * (2 + 34 / 32 + 2), flops=4.0 * T * width)
    if kind == "load":
        return dict(bytes=2.0 * (T + sum(start)) * width * (34 / 32 + 2), flops=2.0 * (T + sum(start)) * width)
    w, keys, seen = case["window"], 0, 0
    for a, n in zip(start, new):
        if n == 0:
            continue
        full = max(0, min(n, a + n - w + 1)) if w else 0  # queries that see w keys
        part = n - full
        keys += full * w + part * a + part * (part + 1) // 2
        seen += min(a + n, w + n - 1) if w else a + n
    row = width * (2 if kind == "packed" else 34 / 32)
    return dict(bytes=4.0 * T * H * hd + 2.0 * seen * row, flops=4.0 * hd * H * keys)


# ---- the same in 64 bits ----

def exact(case, seed):
    i = _inputs(case, seed)
    start, new = _lens(case)
    kind = case["kind"]
    if kind == "verify":
        return _exact_verify(case, i, new)
    H, Hk, hd = HEADS[case["heads"]]

    def where(s, first, upto):
        p = np.arange(first, upto)
        return torch.from_numpy(i["table"][s, p // case["page"]].astype(np.int64) * case["page"] + p % case["page"]).cuda()

    if kind == "store":
        out = {}
        at = torch.cat([where(s, a, a + m) for s, (a, m) in enumerate(zip(start, new))])
        for n in ("k", "v"):
            out[n], d = _exact_store(i[n])
            out[n + "_cache_scales"] = torch.zeros((i["pages"] * case["page"], Hk * hd // 32), dtype=torch.float64, device="cuda")
            out[n + "_cache_scales"][at] = d
        return out

    def values(cache, rows):
        blocks = cache[rows]
        scale = blocks[:, :, 0:2].contiguous().view(torch.float16).double()
        return (blocks[:, :, 2:].contiguous().view(torch.int8).double() * scale).reshape(rows.numel(), Hk, hd)

    if kind == "load":
        return {n: torch.cat([values(i[n + "_cache"], where(s, 0, a + m)).flatten(1) for s, (a, m) in enumerate(zip(start, new))])
                for n in ("k", "v")}
    out = torch.empty((sum(new), H, hd), dtype=torch.float64, device="cuda")
    off = 0
    for s, (a, n) in enumerate(zip(start, new)):
        if kind == "paged":
            rows = where(s, 0, a + n)
            k, v = values(i["k_cache"], rows), values(i["v_cache"], rows)
        else:
            k, v = i["k"][off:off + n].double(), i["v"][off:off + n].double()
        for h in range(H):
            kh, vh = k[:, h // (H // Hk)].T.contiguous(), v[:, h // (H // Hk)].contiguous()
            for t in range(0, n, 2048):
                e = min(n, t + 2048)
                score = (i["q"][off + t:off + e, h].double() @ kh) * hd ** -0.5
                query = torch.arange(a + t, a + e, device="cuda").unsqueeze(1)
                key = torch.arange(a + n, device="cuda").unsqueeze(0)
                seen = key <= query
                if case["window"]:
                    seen &= key > query - case["window"]
                out[off + t:off + e, h] = torch.softmax(score.masked_fill(~seen, -math.inf), 1) @ vh
        off += n
    return out


def _exact_store(x):
    """The format's own steps (each of its 32-bit divisions and products is the 64-bit one rounded)."""
    b = x.double().reshape(x.shape[0], -1, 32)
    d = (b.abs().amax(-1, keepdim=True) / 127).float().double()
    inv = torch.where(d > 0, (1 / torch.where(d > 0, d, 1.0)).float().double(), 0.0)
    y = (b * inv).float().double()
    code = (y.sign() * (y.abs() + 0.5).floor()).clamp(-128, 127)
    return (code * d.half().double()).reshape(x.shape[0], -1), d[..., 0]


def _exact_verify(case, i, new):
    accepted, answer, off = [], [], 0
    for s, n in enumerate(new):
        got, a = [], 0
        for r in range(n):
            x = i["logits"][off + r].double()
            if case["temp"] == 0:
                best = int((x == x.max()).nonzero()[-1])
                if r < n - 1 and int(i["tokens"][off + r + 1]) == best:
                    got.append(best)
                    a += 1
                    continue
                got.append(best)
                break
            p = torch.softmax(x / case["temp"], 0)
            if r < n - 1:
                u = float(i["u"][off + r])
                d = int(i["tokens"][off + r + 1])
                q = None if i["probs"] is None else i["probs"][off - s + r].double()
                if u * (1.0 if q is None else float(q[d])) < float(p[d]):
                    got.append(d)
                    a += 1
                    continue
                if q is None:
                    rest = p.clone()
                    rest[d] = 0.0
                else:
                    rest = torch.clamp(p - q, min=0.0)
                p = rest if float(rest.sum()) > 0 else p
            total = torch.cumsum(p, 0)
            above = (total > float(i["u"][off + n - 1]) * float(total[-1])).nonzero()
            got.append(int(above[0]) if above.numel() else int((p > 0).nonzero()[-1]))
            break
        accepted.append(a)
        answer += got + [-1] * (n - len(got))
        off += n
    return dict(accepted=torch.tensor(accepted, dtype=torch.int32), answer=torch.tensor(answer, dtype=torch.int32))
