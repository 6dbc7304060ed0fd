"""GPU: a step of several sequences (paged store and read-back, attention over the pages and
of packed prompts, checks of drafted tokens) against 64-bit forms (tests/step_reference.py)."""
import numpy as np
import pytest

from sulimo_amd import hip
from tests import step_reference as R

pytestmark = pytest.mark.gpu

HEADS = [(12, 2, 128), (24, 8, 128), (4, 2, 64), (3, 3, 64), (5, 1, 128), (40, 10, 64), (16, 1, 64)]


def up(ctx, a):
    return hip.HipBuffer.from_host(ctx, np.ascontiguousarray(a), True)


def make_table(rng, start, new, page, spare=2):
    """(page table, pages): the sequences' pages in mixed order."""
    need = [-(-(a + b) // page) for a, b in zip(start, new)]
    pages = sum(need) + spare
    order = rng.permutation(pages)
    table = np.zeros((len(new), max(max(need), 1)), np.uint32)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k]
        at += k
    return table, pages


def garbage_cache(rng, rows, width):
    """A cache whose every row that a call must not use holds NaN scales and wild codes."""
    c = rng.integers(0, 256, (rows, width // 32, 34)).astype(np.uint8)
    c[..., :2] = np.array([np.nan], np.float16).view(np.uint8)
    return c.reshape(rows, -1)


def randn16(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


class Step:
    """A batch with a filled cache: keys and values of all cached positions and the new ones."""

    def __init__(self, ctx, rng, heads, start, new, page, window=0, spikes=True):
        self.H, self.Hk, self.hd = heads
        self.ctx, self.start, self.new, self.page, self.window = ctx, start, new, page, window
        width = self.Hk * self.hd
        self.table, self.pages = make_table(rng, start, new, page)
        self.rows = sum(new)
        self.q = randn16(rng, self.rows, self.H, self.hd)
        self.kv = []  # per tensor: f16 rows of every sequence's positions
        for which in range(2):
            seqs = []
            for s, (a, n) in enumerate(zip(start, new)):
                x = randn16(rng, a + n, width)
                if which and spikes and n > 1:  # values that show at once if a query sees the position behind its own
                    x[a + 1:] *= np.float16(50)
                seqs.append(x)
            self.kv.append(seqs)
        self.cache = [garbage_cache(rng, self.pages * page, width) for _ in range(2)]
        self.values = []
        for which in range(2):
            vals = []
            for s, x in enumerate(self.kv[which]):
                if len(x):
                    r, _ = R.quantize(x)
                    self.cache[which][R.slots(self.table[s], page, 0, len(x))] = r
                    vals.append(R.dequantize(r))
                else:
                    vals.append(np.zeros((0, width)))
            self.values.append(vals)
        self.batch = hip.SeqBatch(ctx, self.H, self.Hk, self.hd, window, page, self.pages)
        self.batch.set(new, start, self.table)

    def attend(self, out=None):
        kb, vb, qb = up(self.ctx, self.cache[0]), up(self.ctx, self.cache[1]), up(self.ctx, self.q)
        ob = out or hip.HipBuffer.from_host(self.ctx, np.full((self.rows + 3, self.H, self.hd), 7, np.float16))
        hip.enqueue_attention_paged(self.ctx, self.batch, qb, kb, vb, ob)
        return ob.download(np.float16, (self.rows + 3, self.H, self.hd))

    def reference(self):
        out, bound, off = [], [], 0
        for s, (a, n) in enumerate(zip(self.start, self.new)):
            k, v = (self.values[w][s].reshape(a + n, self.Hk, self.hd) for w in range(2))
            o, b = R.attention(self.q[off:off + n], k, v, a, self.window)
            out.append(o)
            bound.append(b)
            off += n
        return np.concatenate(out), np.concatenate(bound)


def check(got, want, bound):
    err = np.abs(got.astype(np.float64) - want)
    worst = np.unravel_index(np.argmax(err / bound), err.shape) if err.size else None
    assert np.all(err <= bound), (worst, got[worst], want[worst], bound[worst])


# ---- the cache ----

CACHE = [([0], [1], 16), ([5, 0, 130], [1, 70, 3], 16), ([0, 64, 1], [65, 1, 0], 64), ([17, 3], [40, 9], 7), ([2, 0], [3, 2], 1),
         ([300], [260], 256)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("start,new,page", CACHE)
@pytest.mark.parametrize("values", [False, True])
def test_store(ctx, heads, start, new, page, values):
    rng = np.random.default_rng([heads[0], page, sum(new)])
    width = heads[1] * heads[2]
    table, pages = make_table(rng, start, new, page)
    x = [randn16(rng, sum(new), width) * np.float16(3) for _ in range(2)]
    for a in x:  # a block of zeros, of one sign, of the type's largest and smallest
        b = a.reshape(-1, 32)
        b[0] = 0
        b[1] = np.abs(b[1])
        b[len(b) // 2] = 65504
        b[-1] = 6e-8
    old = [rng.integers(0, 256, (pages * page, width // 32 * 34)).astype(np.uint8) for _ in range(2)]
    want = [o.copy() for o in old]
    at = np.concatenate([R.slots(table[s], page, a, a + n) for s, (a, n) in enumerate(zip(start, new))])
    ref = [R.quantize(a) for a in x]
    for w in range(2):
        want[w][at] = ref[w][0]
    batch = hip.SeqBatch(ctx, *heads, page_size=page, n_pages=pages)
    batch.set(new, start, table)
    cache = [up(ctx, o) for o in old]
    out = [up(ctx, np.full((sum(new) + 2, width), 9, np.float16)) for _ in range(2)] if values else [None, None]
    hip.enqueue_kv_store_paged(ctx, batch, up(ctx, x[0]), up(ctx, x[1]), *cache, *out)
    for w in range(2):
        assert np.array_equal(cache[w].download(np.uint8, old[w].shape), want[w])
        if values:
            got = out[w].download(np.float16, (sum(new) + 2, width))
            assert np.array_equal(got[:-2].view(np.uint16), ref[w][1].view(np.uint16)) and np.all(got[-2:] == 9)


def test_store_writes_the_rings_bytes(ctx):
    """Pages in order are the ring: both entry points leave the same bytes."""
    rng = np.random.default_rng(3)
    n, width, page, pages, start = 70, 256, 16, 9, 37
    x = randn16(rng, n, width)
    table = np.arange(pages, dtype=np.uint32)[None]
    batch = hip.SeqBatch(ctx, 12, 2, 128, page_size=page, n_pages=pages)
    batch.set([n], [start], table)
    zero = np.zeros((page * pages, width // 32 * 34), np.uint8)
    k, v, ring = up(ctx, zero), up(ctx, zero), up(ctx, zero)
    xb = up(ctx, x)
    hip.enqueue_kv_store_paged(ctx, batch, xb, xb, k, v)
    hip.enqueue_kv_store(ctx, xb, ring, start, page * pages, width // 32, n)
    want = ring.download(np.uint8, zero.shape)
    assert np.array_equal(k.download(np.uint8, zero.shape), want) and np.array_equal(v.download(np.uint8, zero.shape), want)


def test_store_of_what_is_not_finite_writes_the_rings_bytes(ctx):
    """Blocks with infinities and NaN among their values, and with nothing else."""
    rng = np.random.default_rng(31)
    n, width = 16, 128
    x = randn16(rng, n, width)
    x[1, 5], x[2, 40], x[3, 70], x[4, 3] = np.inf, -np.inf, np.nan, np.inf
    x[4, 4], x[5, :32], x[6, 32:64], x[7] = np.nan, np.nan, np.inf, -np.inf
    batch = hip.SeqBatch(ctx, 2, 1, 128, page_size=n, n_pages=1)
    batch.set([n], [0], [[0]])
    zero = np.zeros((n, width // 32 * 34), np.uint8)
    k, v, ring, xb = up(ctx, zero), up(ctx, zero), up(ctx, zero), up(ctx, x)
    hip.enqueue_kv_store_paged(ctx, batch, xb, xb, k, v)
    hip.enqueue_kv_store(ctx, xb, ring, 0, n, width // 32, n)
    assert np.array_equal(k.download(np.uint8, zero.shape), ring.download(np.uint8, zero.shape))


def test_store_in_place(ctx):
    """k_values and v_values may be k and v."""
    rng = np.random.default_rng(32)
    n, width = 77, 192
    x = [randn16(rng, n, width) for _ in range(2)]
    batch = hip.SeqBatch(ctx, 3, 3, 64, page_size=16, n_pages=5)
    batch.set([n], [0], [[3, 1, 0, 4, 2]])
    kv, cache = [up(ctx, a) for a in x], [hip.HipBuffer.device_only(ctx, 80 * width // 32 * 34) for _ in range(2)]
    hip.enqueue_kv_store_paged(ctx, batch, *kv, *cache, *kv)
    for b, a in zip(kv, x):
        assert np.array_equal(b.download(np.float16, a.shape).view(np.uint16), R.quantize(a)[1].view(np.uint16))


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("start,new,page", CACHE)
def test_load(ctx, heads, start, new, page):
    rng = np.random.default_rng([heads[0], page, 5])
    st = Step(ctx, rng, heads, start, new, page)
    width = heads[1] * heads[2]
    n = sum(start) + sum(new)
    out = [up(ctx, np.full((n + 2, width), 9, np.float16)) for _ in range(2)]
    hip.enqueue_kv_load_paged(ctx, st.batch, up(ctx, st.cache[0]), up(ctx, st.cache[1]), *out)
    for w in range(2):
        got = out[w].download(np.float16, (n + 2, width))
        want = np.concatenate(st.values[w]).astype(np.float16)
        assert np.array_equal(got[:-2].view(np.uint16), want.view(np.uint16)) and np.all(got[-2:] == 9)


# ---- attention over the pages ----

STEPS = [
    ([0], [1], 16, 0), ([31], [1], 16, 0), ([32], [1], 48, 0), ([63, 64, 65], [1, 1, 1], 64, 0), ([1000], [1], 7, 0),
    ([700, 3, 0, 129], [1, 5, 1, 2], 32, 0), ([10, 0, 5], [0, 3, 0], 16, 0), ([0], [33], 16, 0), ([5], [70], 100, 0),
    ([400, 2], [40, 1], 64, 0), ([0, 190], [130, 64], 1, 0), ([90], [200], 256, 0),
    ([500], [1], 16, 1), ([500, 20], [1, 4], 16, 33), ([300], [50], 32, 64), ([0, 77], [90, 1], 16, 40), ([200], [9], 16, 4000),
    ([300], [270], 32, 64), ([500, 3, 90], [300, 1, 5], 16, 0),
]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("start,new,page,window", STEPS)
def test_attention_paged(ctx, heads, start, new, page, window):
    st = Step(ctx, np.random.default_rng([heads[0], page, window, sum(new)]), heads, start, new, page, window)
    got = st.attend()
    want, bound = st.reference()
    check(got[:-3], want, bound)
    assert np.all(got[-3:] == 7)  # rows behind the last sequence


@pytest.mark.parametrize("heads", [(12, 2, 128), (24, 8, 128), (4, 2, 64)])
@pytest.mark.parametrize("start,new,page,window", [([9000], [1], 64, 0), ([5000, 100, 3000], [1, 1, 1], 16, 0), ([2500], [70], 64, 0),
                                                   ([3000, 2000], [5, 3], 48, 1500)])
def test_attention_paged_long(ctx, heads, start, new, page, window):
    st = Step(ctx, np.random.default_rng(7), heads, start, new, page, window, spikes=False)
    check(st.attend()[:-3], *st.reference())


def test_attention_paged_repeats_bit_for_bit(ctx):
    st = Step(ctx, np.random.default_rng(8), (24, 8, 128), [3000, 40, 700], [1, 5, 90], 64, 0)
    a, b = st.attend(), st.attend()
    assert np.array_equal(a.view(np.uint16), b.view(np.uint16))


@pytest.mark.parametrize("heads", [(24, 8, 128), (4, 2, 64)])
def test_a_chunk_is_as_near_as_its_tokens_alone(ctx, heads):
    """A chunk whose part of the cache is read back, and the same rows eight at a time, which read it
    directly: both round values and results to f16 and nothing else, so their errors are alike."""
    start, n = 700, 320
    st = Step(ctx, np.random.default_rng(36), heads, [start], [n], 64, 0, spikes=False)
    want, _ = st.reference()
    whole = st.attend()[:n]
    q, parts = st.q, []
    for t in range(0, n, 8):
        st.batch.set([8], [start + t], st.table)
        st.q, st.rows = q[t:t + 8], 8
        parts.append(st.attend()[:8])
    rms = [np.sqrt(np.mean((x.astype(np.float64) - want) ** 2)) for x in (whole, np.concatenate(parts))]
    assert rms[0] <= 1.2 * rms[1] and rms[1] <= 1.2 * rms[0]


def test_attention_hides_what_is_not_finite(ctx):
    """A later token's keys and values that are NaN or infinite stay out of earlier tokens' sums."""
    for heads in [(12, 2, 128), (4, 2, 64)]:
        for start, n in (([40], 6), ([20], 100), ([20], 300)):
            st = Step(ctx, np.random.default_rng(9), heads, start, [n], 16, 0, spikes=False)
            bad = R.slots(st.table[0], 16, start[0] + n - 1, start[0] + n)
            for w, code in ((0, np.nan), (1, np.inf)):
                st.cache[w][bad] = garbage_cache(np.random.default_rng(1), 1, heads[1] * heads[2])
                st.cache[w].reshape(-1, heads[1] * heads[2] // 32, 34)[bad, :, :2] = np.array([code], np.float16).view(np.uint8)
            got = st.attend()
            want, bound = st.reference()
            check(got[:n - 1], want[:n - 1], bound[:n - 1])
            assert not np.any(np.isfinite(got[n - 1]))


@pytest.mark.parametrize("page,pages", [(64, 64000), (48, 84000)])
def test_a_cache_past_four_gigabytes(ctx, page, pages):
    """Pages whose bytes lie past 2^32 hold and give what those at the front do, for single tokens, a
    short chunk and one that is read back."""
    rng = np.random.default_rng(33)
    H, Hk, hd = 24, 8, 128
    width, each = Hk * hd, -(-333 // page)
    assert pages * page * (width // 32) * 34 > 1 << 32
    start, new = [0, 0, 0], [260, 300, 333]
    k, v = (randn16(rng, sum(new), width) for _ in range(2))
    kv = up(ctx, k), up(ctx, v)
    steps = [([259, 290, 250], [1, 10, 83]), (start, new)]
    q = [randn16(rng, sum(n), H, hd) for _, n in steps]
    cache = [hip.HipBuffer.device_only(ctx, pages * page * (width // 32) * 34) for _ in range(2)]
    answers = []
    for first in (0, pages - 3 * each):
        table = first + np.arange(3 * each, dtype=np.uint32).reshape(3, each)[:, ::-1]
        batch = hip.SeqBatch(ctx, H, Hk, hd, 0, page, pages)
        batch.set(new, start, table)
        hip.enqueue_kv_store_paged(ctx, batch, *kv, *cache)
        out = [hip.HipBuffer.device_only(ctx, k.nbytes) for _ in range(2)]
        hip.enqueue_kv_load_paged(ctx, batch, *cache, *out)
        got = [b.download(np.float16, k.shape) for b in out]
        for x, y in zip(got, (k, v)):
            assert np.array_equal(x.view(np.uint16), R.quantize(y)[1].view(np.uint16))
        for (st, n), x in zip(steps, q):
            batch.set(n, st, table)
            o = hip.HipBuffer.device_only(ctx, x.nbytes)
            hip.enqueue_attention_paged(ctx, batch, up(ctx, x), *cache, o)
            got.append(o.download(np.float16, x.shape))
        answers.append(got)
        batch.release()
    for a, b in zip(*answers):
        assert np.array_equal(a.view(np.uint16), b.view(np.uint16))
    assert np.isfinite(answers[0][2]).all() and np.abs(answers[0][3]).max() > 0


@pytest.mark.parametrize("new", [1, 20, 90])
def test_pages_behind_the_window_may_stand_for_anything(ctx, new):
    """A table's entries behind the window may all name one page that another sequence filled."""
    rng = np.random.default_rng([34, new])
    x = Step(ctx, rng, (24, 8, 128), [700, 300], [new, new], 16, window=100)
    want = x.attend()
    table = x.table.copy()
    for s, a in enumerate(x.start):
        table[s, :(a - 100 + 1) // 16] = x.pages - 1  # a spare page: NaN scales and wild codes
    assert not (table == x.table).all()
    x.batch.set(x.new, x.start, table)
    assert np.array_equal(x.attend().view(np.uint16), want.view(np.uint16))
    check(want[:-3], *x.reference())


def test_prefills_and_steps_in_turn(ctx):
    """A prefill of one sequence and steps of several share the context's workspace, and neither
    changes what the other gives."""
    from sulimo_amd import synthetic as S
    cfg = S.ModelConfig(2, 256, 512, 4, 2, 64, 64, 512, 1e6, 1e-6, 1)
    dm = hip.DeviceModel(ctx, S.make_model(cfg, 7), capacity=64, max_n=16)
    toks = S.random_tokens(8, 32, cfg.vocab)
    steps = [Step(ctx, np.random.default_rng([37, i]), (4, 2, 64), start, new, 16) for i, (start, new) in
             enumerate([([900], [1]), ([50, 700], [300, 4]), ([2000] * 30, [9] * 30)])]
    alone = [x.attend() for x in steps]

    def prefill(between):
        out = []
        for at in (0, 16):
            dm.embed(toks[at:at + 16])
            dm.execute_prefill_ubatch(at, 16)
            out.append(dm.logits().copy())
            between(at)
        return out

    want = prefill(lambda at: None)
    for turn in range(3):
        got = []
        logits = prefill(lambda at: got.extend(x.attend() for x in steps))
        assert all(np.array_equal(a, b) for a, b in zip(logits, want)), turn
        assert all(np.array_equal(a.view(np.uint16), b.view(np.uint16)) for a, b in zip(got, alone + alone)), turn
    dm.release()


def test_contexts_and_batches_that_grow_and_shrink(ctx):
    """Two contexts in turn without a wait, each with a batch that grows, shrinks and grows."""
    other = hip.HipContext.new(0)
    jobs, outs = [], []
    for i, (n_seqs, new) in enumerate([(1, 1), (40, 3), (2, 100), (1, 1), (64, 1), (3, 400)]):
        for c in (ctx, other):
            jobs.append(Step(c, np.random.default_rng([35, i]), (4, 2, 64), [(37 * j) % 900 for j in range(n_seqs)],
                             [new] * n_seqs, 32))
    own = {id(c): hip.SeqBatch(c, 4, 2, 64, 0, 32, max(j.pages for j in jobs)) for c in (ctx, other)}
    for j in jobs:
        rows = max(k.pages for k in jobs) * 32
        cache = [up(j.ctx, np.concatenate([y, np.zeros((rows - len(y), y.shape[1]), np.uint8)])) for y in j.cache]
        b = own[id(j.ctx)]
        b.set(j.new, j.start, j.table)
        o = hip.HipBuffer.device_only(j.ctx, j.q.nbytes)
        hip.enqueue_attention_paged(j.ctx, b, up(j.ctx, j.q), *cache, o)
        outs.append(o)
    got = [o.download(np.float16, j.q.shape) for o, j in zip(outs, jobs)]
    for i in range(0, len(jobs), 2):
        assert np.array_equal(got[i].view(np.uint16), got[i + 1].view(np.uint16))
        check(got[i], *jobs[i].reference())
    own[id(other)].release()
    for j in jobs:
        j.batch.release()
    del outs, jobs
    other.release()


def test_two_batches_take_turns_without_a_wait(ctx):
    """Work queued on one batch keeps the sequences it was queued with, also when set comes before it ran."""
    rng = np.random.default_rng(10)
    a = Step(ctx, rng, (12, 2, 128), [900, 5], [1, 40], 16)
    b = Step(ctx, rng, (24, 8, 128), [50] * 20, [1] * 20, 32)
    bufs = {}
    for name, st in (("a", a), ("b", b)):
        bufs[name] = (up(ctx, st.q), up(ctx, st.cache[0]), up(ctx, st.cache[1]))
    outs = []
    for turn in range(3):
        for name, st in (("a", a), ("b", b)):
            o = hip.HipBuffer.device_only(ctx, (st.rows + 3) * st.H * st.hd * 2)
            hip.enqueue_attention_paged(ctx, st.batch, *bufs[name], o)
            outs.append((st, o))
        # the same batch with other sequences: two of the first one's, the other way round
        a.batch.set([1], [5], a.table[:1])
        a.batch.set(a.new, a.start, a.table)
    for st, o in outs:
        check(o.download(np.float16, (st.rows, st.H, st.hd)), *st.reference())


# ---- packed prompts ----

@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("new,window", [([1], 0), ([2, 1, 0, 3], 0), ([31, 32, 33], 0), ([64, 65], 0), ([130], 0), ([300, 7], 0),
                                        ([200, 5], 1), ([257], 64), ([100, 140], 50)])
def test_attention_packed(ctx, heads, new, window):
    H, Hk, hd = heads
    rng = np.random.default_rng([H, window, sum(new)])
    rows = sum(new)
    q, k, v = randn16(rng, rows, H, hd), randn16(rng, rows, Hk, hd), randn16(rng, rows, Hk, hd)
    v[1::2] *= np.float16(30)
    batch = hip.SeqBatch(ctx, H, Hk, hd, window)
    batch.set(new)
    ob = up(ctx, np.full((rows + 3, H, hd), 7, np.float16))
    hip.enqueue_attention_packed(ctx, batch, up(ctx, q), up(ctx, k), up(ctx, v), ob)
    got = ob.download(np.float16, (rows + 3, H, hd))
    off = 0
    for n in new:
        at = slice(off, off + n)
        check(got[at], *R.attention(q[at], k[at].astype(np.float64), v[at].astype(np.float64), 0, window))
        off += n
    assert np.all(got[rows:] == 7)


def test_attention_packed_hides_what_is_not_finite(ctx):
    """NaN and infinities of later tokens, and of the next sequence, stay out of a token's sum."""
    for H, Hk, hd in [(12, 2, 128), (4, 2, 64)]:
        rng = np.random.default_rng(11)
        new = [90, 70]
        q, k, v = randn16(rng, 160, H, hd), randn16(rng, 160, Hk, hd), randn16(rng, 160, Hk, hd)
        k[80], v[80] = np.nan, np.inf
        v[90 + 60, :, ::2] = np.nan
        v[90 + 60, :, 1::2] = -np.inf
        batch = hip.SeqBatch(ctx, H, Hk, hd)
        batch.set(new)
        ob = hip.HipBuffer.device_only(ctx, 160 * H * hd * 2)
        hip.enqueue_attention_packed(ctx, batch, up(ctx, q), up(ctx, k), up(ctx, v), ob)
        got = ob.download(np.float16, (160, H, hd))
        for a, n, bad in ((0, 90, 80), (90, 70, 60)):
            kk, vv = k[a:a + n].astype(np.float64), v[a:a + n].astype(np.float64)
            check(got[a:a + bad], *R.attention(q[a:a + bad], kk, vv, 0, 0))
            assert not np.any(np.isfinite(got[a + bad:a + n]))
        assert np.all(got[150:, :, 1::2] == -np.inf) and np.all(np.isnan(got[150:, :, ::2]))


def test_stored_values_serve_the_packed_form(ctx):
    """A prompt's stored values through the packed form, and its pages through the paged form:
    both are within their bounds of the same sum."""
    rng = np.random.default_rng(12)
    new = [70, 200, 1]
    st = Step(ctx, rng, (24, 8, 128), [0] * 3, new, 16)
    k, v = (np.concatenate(st.kv[w]) for w in range(2))
    cache = [up(ctx, np.zeros_like(st.cache[0])) for _ in range(2)]
    vals = [hip.HipBuffer.device_only(ctx, k.nbytes) for _ in range(2)]
    outs = [hip.HipBuffer.device_only(ctx, st.q.nbytes) for _ in range(2)]
    qb = up(ctx, st.q)
    hip.enqueue_kv_store_paged(ctx, st.batch, up(ctx, k), up(ctx, v), *cache, *vals)
    hip.enqueue_attention_packed(ctx, st.batch, qb, *vals, outs[0])
    hip.enqueue_attention_paged(ctx, st.batch, qb, *cache, outs[1])
    want, bound = st.reference()
    for o in outs:
        check(o.download(np.float16, st.q.shape), want, bound)


# ---- drafted tokens ----

def run_verify(ctx, logits, tokens, probs, u, n_new, temperature):
    V = logits.shape[1]
    batch = hip.SeqBatch(ctx)
    batch.set(n_new)
    acc = up(ctx, np.full(len(n_new) + 1, 77, np.int32))
    ans = up(ctx, np.full(sum(n_new) + 1, 77, np.int32))
    hip.enqueue_verify_drafts(ctx, batch, up(ctx, logits), up(ctx, tokens.astype(np.int32)), None if probs is None else up(ctx, probs),
                              None if u is None else up(ctx, u.astype(np.float32)), V, temperature, acc, ans)
    a, r = acc.download(np.int32, len(n_new) + 1), ans.download(np.int32, sum(n_new) + 1)
    assert a[-1] == 77 and r[-1] == 77
    return a[:-1], r[:-1]


def drafted(rng, n_new, V, point, noise=0.5):
    rows = sum(n_new)
    logits = (2 * rng.standard_normal((rows, V))).astype(np.float32)
    tokens = rng.integers(0, V, rows).astype(np.int32)
    judge = np.concatenate([np.arange(o, o + n - 1) for o, n in zip(np.cumsum([0] + n_new[:-1]), n_new)]).astype(int)
    x = logits[judge] + noise * rng.standard_normal((len(judge), V))
    probs = np.exp(x - x.max(-1, keepdims=True)) if len(judge) else x
    probs = (probs / probs.sum(-1, keepdims=True)).astype(np.float32) if len(judge) else probs.astype(np.float32)
    for i, r in enumerate(judge):
        tokens[r + 1] = probs[i].argmax() if point else rng.choice(V, p=probs[i].astype(np.float64) / probs[i].astype(np.float64).sum())
    return logits, tokens, None if point or not len(judge) else probs, rng.random(rows).astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 63, 64, 1000, 4097, 32000, 70001])
@pytest.mark.parametrize("n_new", [[1], [5], [1, 4, 9, 2], [3] * 30])
@pytest.mark.parametrize("point,temperature", [(False, 1.0), (False, 0.4), (True, 1.3), (True, 0.0)])
def test_verify(ctx, V, n_new, point, temperature):
    rng = np.random.default_rng([V, len(n_new), sum(n_new), point])
    args = drafted(rng, n_new, V, point)
    got = run_verify(ctx, *args, n_new, temperature)
    want = R.verify(*args, n_new, temperature)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_verify_follows_every_branch(ctx):
    """Rows made so that drafts are all accepted, refused at each place, and refused with nothing left."""
    rng = np.random.default_rng(13)
    V, n_new = 501, [4] * 6
    logits, tokens, probs, u = drafted(rng, n_new, V, False, noise=0.0)
    u[:] = 0.999
    for s in range(4):  # sequence s: draft s is one the target hardly gives
        if s < 3:
            tokens[4 * s + s + 1] = 7
            logits[4 * s + s, 7] = -50.0
    u[4 * 3 + 3] = 0.0          # the first token with any mass
    u[4 * 4 + 3] = 1.0 - 2**-24  # the last ones
    # q = p of a row with one possible token: refused only by an id outside the vocabulary, nothing is left of p - q
    logits[4 * 5] = -np.inf
    logits[4 * 5, 9] = 3.0
    probs[3 * 5] = 0.0
    probs[3 * 5, 9] = 1.0
    tokens[4 * 5 + 1] = V
    got = run_verify(ctx, logits, tokens, probs, u, n_new, 1.0)
    want = R.verify(logits, tokens, probs, u, n_new, 1.0)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    assert list(want[0][:4]) == [0, 1, 2, 3] and want[1][4 * 5] == 9


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_verify_of_odd_logits(ctx, temperature):
    """Rows with NaN, infinities, equal greatest entries, nothing at all; ids and probabilities out of range."""
    V, n_new = 300, [2] * 8
    rng = np.random.default_rng(14)
    logits, tokens, probs, u = drafted(rng, n_new, V, False)
    logits[0] = -np.inf            # nothing to choose from
    logits[2] = np.nan
    logits[4, 5:] = np.nan
    logits[6, [3, 200, 299]] = np.inf
    logits[8] = -3.4e38            # all equal, the type's lowest
    logits[10, :] = -np.inf
    logits[10, 17] = -np.inf
    logits[11] = -np.inf
    tokens[13] = -5
    probs[7] = np.nan
    probs[6, ::2] = -1.0
    u[14] = np.nan
    u[9] = 2.0
    u[5] = -1.0
    got = run_verify(ctx, logits, tokens, probs, u, n_new, temperature)
    want = R.verify(logits, tokens, probs, u, n_new, temperature)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_verify_keeps_the_targets_distribution(ctx):
    """Drafted or not, a position's token is distributed as the target's: 20000 sequences of one
    draft each, 8 tokens; the counts are within 5 sigma of n p."""
    rng = np.random.default_rng(15)
    V, n = 8, 20000
    logits = np.tile(rng.standard_normal((2, V)).astype(np.float32), (n, 1))
    q = rng.random(V) + 0.05
    q = (q / q.sum()).astype(np.float32)
    tokens = np.zeros(2 * n, np.int32)
    tokens[1::2] = rng.choice(V, n, p=q.astype(np.float64) / q.astype(np.float64).sum())
    _, ans = run_verify(ctx, logits, tokens, np.tile(q, (n, 1)), rng.random(2 * n).astype(np.float32), [2] * n, 1.0)
    p = np.exp(logits[0].astype(np.float64))
    p /= p.sum()
    count = np.bincount(ans[0::2], minlength=V)
    assert np.all(np.abs(count - n * p) <= 5 * np.sqrt(n * p * (1 - p)))


# ---- a step as it is run, and refusals ----

def test_steps_of_a_conversation(ctx):
    """Prompts, then drafted steps: store, attend, check, and the next step starts behind the
    accepted tokens, writing over the refused ones' rows. Every step's attention and answers
    against the 64-bit forms of what was kept."""
    rng = np.random.default_rng(16)
    H, Hk, hd, page, V, S = 12, 2, 128, 16, 800, 3
    width, pages = Hk * hd, 40
    table = rng.permutation(pages)[:S * 12].reshape(S, 12).astype(np.uint32)
    cache = [up(ctx, garbage_cache(rng, pages * page, width)) for _ in range(2)]
    batch = hip.SeqBatch(ctx, H, Hk, hd, 0, page, pages)
    kept = [[np.zeros((0, width)) for _ in range(S)] for _ in range(2)]  # values the cache stands for
    lens = [20, 37, 5]
    for turn in range(4):
        start = [len(kept[0][s]) for s in range(S)]
        batch.set(lens, start, table)
        rows = sum(lens)
        q, kv = randn16(rng, rows, H, hd), [randn16(rng, rows, width) for _ in range(2)]
        logits, tokens, probs, u = drafted(rng, lens, V, False)
        out, acc, ans = (hip.HipBuffer.device_only(ctx, n) for n in (q.nbytes, 4 * S, 4 * rows))
        hip.enqueue_kv_store_paged(ctx, batch, up(ctx, kv[0]), up(ctx, kv[1]), *cache)
        hip.enqueue_attention_paged(ctx, batch, up(ctx, q), *cache, out)
        hip.enqueue_verify_drafts(ctx, batch, up(ctx, logits), up(ctx, tokens), None if probs is None else up(ctx, probs),
                                  up(ctx, u), V, 1.0, acc, ans)
        a, r = acc.download(np.int32, S), ans.download(np.int32, rows)
        want = R.verify(logits, tokens, probs, u, lens, 1.0)
        assert np.array_equal(a, want[0]) and np.array_equal(r, want[1])
        got, off = out.download(np.float16, q.shape), 0
        for s, n in enumerate(lens):
            full = [np.concatenate([kept[w][s], R.dequantize(R.quantize(kv[w][off:off + n])[0])]) for w in range(2)]
            check(got[off:off + n], *R.attention(q[off:off + n], *(x.reshape(-1, Hk, hd) for x in full), start[s], 0))
            stay = n if turn == 0 else int(a[s]) + 1  # a prompt stays whole
            for w in range(2):
                kept[w][s] = full[w][:start[s] + stay]
            off += n
        lens = [5, 5, 3]


def refused(code, f, *a):
    with pytest.raises(hip.HipError) as e:
        f(*a)
    assert e.value.code == code, e.value


def test_refusals(ctx):
    bad = hip.ERR_INVALID_ARGUMENT
    other = hip.HipContext.new(0)
    big = hip.HipBuffer.device_only(ctx, 1 << 20)
    big2, big3, big4 = (hip.HipBuffer.device_only(ctx, 1 << 20) for _ in range(3))
    small = hip.HipBuffer.device_only(ctx, 16)
    b = hip.SeqBatch(ctx, 4, 2, 64, 0, 16, 8)
    refused(bad, hip.enqueue_attention_paged, ctx, b, big, big2, big3, big4)  # no sequences, no pages yet
    b.set([3], [20], [[0, 1]])
    for args in ((small, big2, big3, big4), (big, small, big3, big4), (big, big2, small, big4), (big, big2, big3, small),
                 (None, big2, big3, big4), (big, big2, big3, big)):
        refused(bad, hip.enqueue_attention_paged, ctx, b, *args)
        refused(bad, hip.enqueue_attention_packed, ctx, b, *args)
    refused(bad, hip.enqueue_attention_packed, ctx, b, big, big2, big3, big4)  # cached positions
    refused(bad, hip.enqueue_attention_paged, other, b, big, big2, big3, big4)  # another context
    refused(bad, hip.enqueue_kv_store_paged, ctx, b, big, big2, big3, big3)
    refused(bad, hip.enqueue_kv_store_paged, ctx, b, big, big2, big3, big4, small)
    refused(bad, hip.enqueue_kv_load_paged, ctx, b, big, big2, small, big4)
    refused(bad, hip.enqueue_kv_load_paged, ctx, b, big, big2, big3, big3)
    for args in ((big, big2, big3, big2), (big, big2, big, big4), (big, big2, big3, big4, big2), (big, big2, big3, big4, big3),
                 (big, big2, big3, big4, None, big), (big, big2, big3, big4, big, big)):  # one buffer twice
        refused(bad, hip.enqueue_kv_store_paged, ctx, b, *args)
    for args in ((big, big2, big, big4), (big, big2, big3, big2)):
        refused(bad, hip.enqueue_kv_load_paged, ctx, b, *args)
    for args in ((big, big2, big3, big2), (big, big2, big3, big3)):
        refused(bad, hip.enqueue_attention_paged, ctx, b, *args)
    refused(bad, b.set, [1], [127], [[0] * 7 + [9]])
    hip.enqueue_attention_paged(ctx, b, big, big2, big3, big4)  # a refused set left the sequences as they were
    v = hip.SeqBatch(ctx)
    v.set([2, 1])
    ok = (big, big2, big3, big4, 100, 1.0)
    acc, ans = hip.HipBuffer.device_only(ctx, 8), hip.HipBuffer.device_only(ctx, 12)
    hip.enqueue_verify_drafts(ctx, v, *ok, acc, ans)
    for args in ((small, *ok[1:]), (big, None, *ok[2:]), (big, big2, small, *ok[3:]), (big, big2, big3, None, 100, 1.0),
                 (*ok[:4], 0, 1.0), (*ok[:4], 100, -1.0), (*ok[:4], 100, float("nan")), (*ok[:4], 100, float("inf"))):
        refused(bad, hip.enqueue_verify_drafts, ctx, v, *args, acc, ans)
    refused(bad, hip.enqueue_verify_drafts, ctx, v, *ok, acc, acc)
    for x in (big, big2, big3, big4):
        refused(bad, hip.enqueue_verify_drafts, ctx, v, *ok, x, ans)
        refused(bad, hip.enqueue_verify_drafts, ctx, v, *ok, acc, x)
    refused(bad, hip.enqueue_attention_packed, ctx, v, big, big2, big3, big4)  # no head layout
    v.set([2, 0])
    refused(bad, hip.enqueue_verify_drafts, ctx, v, *ok, acc, ans)
    ctx.wait()
    b.release()
    b.release()
    c = hip.SeqBatch(other, 4, 2, 64, 0, 16, 8)
    h = c.handle
    c.handle = type(h)()
    hip.lib().sulimo_hip_seq_batch_release(h)
    refused(bad, c.set, [1])
    d = hip.SeqBatch(other, 4, 2, 64)
    d.set([2])
    d.release()
    e = hip.SeqBatch(other)
    e.release()
    other.release()
    refused(bad, e.set, [1])  # its context is gone


def test_empty_steps_do_nothing(ctx):
    b = hip.SeqBatch(ctx, 4, 2, 64, 0, 16, 8)
    bufs = [up(ctx, np.full(8 * 16 * 136, 5, np.uint8)) for _ in range(6)]
    for new, start in (([], []), ([0, 0], [0, 0])):
        b.set(new, start, np.zeros((len(new), 1), np.uint32))
        hip.enqueue_kv_store_paged(ctx, b, *bufs[:4])
        hip.enqueue_kv_load_paged(ctx, b, *bufs[:4])
        hip.enqueue_attention_paged(ctx, b, *bufs[:4])
        b.set(new)
        hip.enqueue_attention_packed(ctx, b, *bufs[:4])
        if not new:
            hip.enqueue_verify_drafts(ctx, b, *bufs[:4], 4, 1.0, *bufs[4:])
    for x in bufs:
        assert np.all(x.download(np.uint8, 8 * 16 * 136) == 5)
