"""The operators of a serving step over the paged 8-bit cache (sq_kv_*,
sq_sdpa_paged, sq_verify_draft) against tests/serving_oracle.py.

Stored integers and scales, accepted counts and tokens are compared for
equality: the kernels decide them in 64 bits.  Attention is f32: its bound is
derived at `bounds`.  The cases marked small also run on the CPU emulator
(tests/test_cpu_serving.py).
"""
import threading

import numpy as np
import pytest

import serving_oracle as S

pytestmark = pytest.mark.gpu

sq = pytest.importorskip("sqhip")
from sqhip import ops  # noqa: E402
from sqhip._lib import (KernelError, LLMError, SQ_ERR_ARG, SQ_ERR_SHAPE, SQ_ERR_UNSUPPORTED, lib)  # noqa: E402
from sqhip.ops import DeviceArray  # noqa: E402

PAGE = S.PAGE


def rng(seed):
    return np.random.default_rng(seed)


def dev(a):
    return DeviceArray.from_numpy(a)


class Step:
    """A pool with its oracle, and page tables in no order."""

    def __init__(self, lengths, kv_heads=2, dim=64, half=None, layers=1, seed=0, spare=3):
        self.r = rng(seed)
        half = dim // 2 if half is None else half
        inv = S.inv_freq(half)
        pages = [max(1, -(-n // PAGE)) for n in lengths]
        total = sum(pages) + spare
        free = self.r.permutation(total)
        self.tables = np.zeros((len(lengths), max(pages)), np.uint32)
        for i, n in enumerate(pages):
            self.tables[i, :n], free = free[:n], free[n:]
        self.free = free
        self.kv_heads, self.dim = kv_heads, dim
        self.pool = ops.KvPool(layers, total, kv_heads, dim, inv)
        self.oracle = [S.Cache(total, kv_heads, dim, inv) for _ in range(layers)]

    def rows(self, n, scale=1.0):
        """n new keys and values; a few keys large, so that scales grow."""
        x = self.r.standard_normal((2, n, self.kv_heads * self.dim)).astype(np.float32) * np.float32(scale)
        x[0, self.r.random(n) < 0.2] *= np.float32(3.7)
        x[1, self.r.random(n) < 0.2] *= np.float32(1.9)
        return x

    def append(self, past, new, layer=0, scale=1.0, rotated=False, rows=None):
        k, v = self.rows(int(np.sum(new)), scale) if rows is None else rows
        plan = ops.KvPlan(self.pool, past, new, self.tables)
        ops.kv_append(plan, layer, dev(k), dev(v), rotated=rotated)
        self.oracle[layer].append(past, new, self.tables, k, v, rotated)
        return plan

    def check_cache(self, plan, past, new, layer=0, last=1 << 30):
        n = [min(int(a + b), last) for a, b in zip(past, new)]
        shape = (sum(n), self.kv_heads, self.dim)
        k, v = DeviceArray(shape), DeviceArray(shape)
        ops.kv_read(plan, layer, last, k, v)
        for which, got in ((0, k.numpy()), (1, v.numpy())):
            want = [self.oracle[layer].values(self.tables[i], int(a + b), which, int(a + b) - m)
                    for i, (a, b, m) in enumerate(zip(past, new, n))]
            want = np.concatenate(want) if want else np.zeros(shape, np.float32)
            assert np.array_equal(got, want), ("keys", "values")[which]

    def attend(self, plan, past, new, heads, window=0, sinks=0, layer=0, rotated=False, q=None, scale=1.0):
        n = int(np.sum(new))
        if q is None:
            q = self.r.standard_normal((n, heads * self.dim)).astype(np.float32) * np.float32(scale)
        out = DeviceArray((n, heads * self.dim))
        ops.sdpa_paged(plan, layer, dev(q), out, heads, window=window, sinks=sinks, rotated=rotated)
        want, amp, vmax = S.sdpa(self.oracle[layer], past, new, self.tables, q, heads, window, sinks, rotated)
        close(out.numpy(), want, amp, vmax, self.dim, int(np.max(np.add(past, new))))


def close(got, want, amp, vmax, dim, length):
    """Bounds on an output of f32 attention over exact cached values.

    A score is a sum of dim products: q is rounded to f32 after its rotation
    (2^-24) and taken in two halves of 11 bits (2^-22), each of the sum's
    dim + 8 additions and the scalings rounds (2^-24 of at most amp = sum
    |q k| / sqrt(d)), its distance from the maximum rounds at most 2 amp: the
    weight's exponent is off by at most e = amp (dim + 16) 2^-24, the weight by
    that, by the exponential's and by its own two halves (2^-21).  The output
    is a quotient of sums of weights: 2 (e + 2^-21) vmax, and its own sums round
    once a key at most, 2^-24 length vmax.  Errors that are independent grow
    with the square root of their number: that is the second bound, on the norm."""
    amp, vmax = np.maximum(amp, 1e-30), np.maximum(vmax, 1e-30)
    shape = amp.shape[:2] + (dim,)
    err = np.abs(got.reshape(shape) - want.reshape(shape))
    e = amp * (dim + 16) * 2.0**-24
    assert np.all(err <= vmax * (2 * (e + 2.0**-21) + length * 2.0**-24)), float((err / vmax).max())
    rel = np.linalg.norm(err) / max(np.linalg.norm(want), 1e-30)
    assert rel <= 2 * (amp.max() * np.sqrt(dim + 16) * 2.0**-24 + 2.0**-21), rel


# ---------------------------------------------------------------- the cache

CACHE = [
    ("small", 64, 2, [(0, 1)]),
    ("small", 64, 1, [(0, 64), (0, 65), (0, 0), (0, 130)]),
    ("small", 128, 2, [(0, 63), (0, 100)]),
    ("large", 64, 8, [(0, 1000), (0, 1), (0, 64), (0, 4097)]),
    ("large", 128, 8, [(0, 700), (0, 1500)]),
]


@pytest.mark.parametrize("size,dim,kv_heads,seqs", CACHE)
def test_append_and_read(size, dim, kv_heads, seqs):
    past, new = map(list, zip(*seqs))
    t = Step([a + b for a, b in seqs], kv_heads, dim, seed=dim + len(seqs))
    plan = t.append(past, new)
    t.check_cache(plan, past, new)
    t.check_cache(plan, past, new, last=1)
    t.check_cache(plan, past, new, last=66)


@pytest.mark.parametrize("size,dim", [("small", 64), ("small", 128), ("large", 64)])
def test_growing_scales_and_rejected_rows(size, dim):
    """Rows arrive one or a few at a time, larger ones among them, and the step
    goes back over rejected rows: each state equals the definition's."""
    lens = [70, 140, 64] if size == "small" else [900, 70, 300, 1]
    t = Step([n + 8 for n in lens], 2, dim, seed=3)
    past = [0] * len(lens)
    for step in range(9 if size == "small" else 40):
        new = [min(int(t.r.integers(0, 40 if step < 2 else 6)), n - p) for n, p in zip(lens, past)]
        plan = t.append(past, new, scale=float(np.exp(t.r.normal())))
        t.check_cache(plan, past, new)
        past = [p + max(0, m - int(t.r.integers(0, 3))) for p, m in zip(past, new)]


@pytest.mark.parametrize("half", [0, 1, 20, 32])
def test_partial_rotation_small(half):
    t = Step([90, 5], 2, 64, half=half, seed=half)
    plan = t.append([0, 0], [90, 5])
    t.check_cache(plan, [0, 0], [90, 5])
    t.attend(plan, [0, 0], [90, 5], 4)


def test_far_positions_rotate_in_64_bits_small():
    past, new = [50000 - 3], [9]
    t = Step([50010], 1, 64, seed=5)
    plan = t.append(past, new)
    t.check_cache(plan, past, new, last=9)
    plan = t.append(past, new, rotated=True)
    t.check_cache(plan, past, new, last=9)


def test_zero_and_tiny_rows_small():
    """A page of zeros has scale 0; rows of the smallest magnitudes, and a page
    whose former rows are zeros."""
    t = Step([64, 64, 64], 1, 64, half=0, seed=6)
    k = np.zeros((30, 64), np.float32)
    k[10:20] = 1e-40
    k[20:] = np.float32(3e38)
    plan = t.append([0, 0, 0], [10, 10, 10], rows=(k, k))
    t.check_cache(plan, [0, 0, 0], [10, 10, 10])
    plan = t.append([10, 10, 10], [3, 3, 3], rows=(k[8:17] + 1, k[8:17]))
    t.check_cache(plan, [10, 10, 10], [3, 3, 3])


def test_rows_apart_in_one_buffer_small():
    """q, k and v as the columns of one product's rows, an odd stride, an address that is
    only a multiple of 4, and rows behind the batch that stay as they were."""
    past, new, heads = [3, 0, 65], [2, 0, 3], 4
    t = Step([5, 1, 68], 2, 64, seed=7)
    t.append([0, 0, 0], past)
    qw, kw = heads * 64, 2 * 64
    width = qw + 2 * kw + 3
    buf = t.r.standard_normal((7, width)).astype(np.float32)
    d = dev(buf)

    class At:
        def __init__(self, ptr, size):
            self.ptr, self.size, self.shape = ptr, size, (size,)

    plan = ops.KvPlan(t.pool, past, new, t.tables)
    q, k, v = (At(d.ptr + 4 * o, 5 * n) for o, n in ((1, qw), (1 + qw, kw), (1 + qw + kw, kw)))
    ops.kv_append(plan, 0, k, v, k_stride=width, v_stride=width)
    kk, vv = buf[:5, 1 + qw:1 + qw + kw], buf[:5, 1 + qw + kw:1 + qw + 2 * kw]
    t.oracle[0].append(past, new, t.tables, kk, vv)
    t.check_cache(plan, past, new)
    want, amp, vmax = S.sdpa(t.oracle[0], past, new, t.tables, buf[:5, 1:1 + qw], heads)
    ops.sdpa_paged(plan, 0, q, q, heads, q_stride=width, out_stride=width)  # in place
    got = d.numpy()
    close(got[:5, 1:1 + qw], want, amp, vmax, 64, 68)
    keep = np.ones_like(buf, bool)
    keep[:5, 1:1 + qw] = False
    assert np.array_equal(got[keep], buf[keep])


def test_layers_and_shared_pages_small():
    """Layers are apart; two sequences share the pages of a common prefix."""
    t = Step([64 + 10, 64 + 20], 2, 64, layers=3, seed=8)
    t.tables[1, 0] = t.tables[0, 0]
    for layer in (0, 2):
        t.append([0, 0], [64, 0], layer=layer)
    for layer in (0, 2):
        plan = t.append([64, 64], [10, 20], layer=layer)
        t.check_cache(plan, [64, 64], [10, 20], layer=layer)
        t.attend(plan, [64, 64], [10, 20], 4, layer=layer)
    k, v = DeviceArray((174 - 16, 2, 64)), DeviceArray((174 - 16, 2, 64))
    ops.kv_read(plan, 1, 1 << 20, k, v)
    assert not k.numpy().any() and not v.numpy().any()  # no call wrote layer 1


def test_values_that_are_not_finite_are_reported_small():
    t = Step([80], 2, 64, half=0, seed=9)
    k, v = t.rows(80)
    k[3, 5], k[70, 64], v[3, 0], v[79, 127] = np.inf, np.nan, -np.inf, np.nan
    plan = ops.KvPlan(t.pool, [0], [80], t.tables)
    with pytest.raises(LLMError) as e:
        ops.kv_append(plan, 0, dev(k), dev(v))
    assert e.value.code == SQ_ERR_ARG
    k[3, 4:6], k[70, 64:66], v[3, 0], v[79, 127] = 0, 0, 0, 0  # a key's whole pair
    t.oracle[0].append([0], [80], t.tables, k, v)
    t.check_cache(plan, [0], [80])
    plan = t.append([0], [80])  # the report is not kept
    t.check_cache(plan, [0], [80])


# ---------------------------------------------------------------- attention

SDPA = [
    # size, dim, heads, kv_heads, (past, new) of each sequence, window, sinks
    ("small", 64, 4, 1, [(0, 1)], 0, 0),
    ("small", 64, 4, 2, [(62, 1), (63, 1), (64, 1), (0, 0), (200, 1)], 0, 0),
    ("small", 64, 8, 2, [(0, 17), (130, 5)], 0, 0),
    ("small", 64, 3, 3, [(1, 70)], 0, 0),
    ("small", 64, 6, 1, [(60, 9), (300, 1)], 0, 0),
    ("small", 128, 4, 2, [(0, 66), (127, 2)], 0, 0),
    ("small", 64, 4, 2, [(300, 1), (10, 4), (63, 3)], 64, 0),
    ("small", 64, 4, 2, [(300, 1), (250, 40)], 100, 4),
    ("small", 64, 2, 2, [(0, 140)], 1, 0),
    ("small", 64, 2, 2, [(0, 140)], 5, 70),
    ("small", 64, 2, 1, [(200, 3)], 1 << 31, 1 << 31),
    ("small", 128, 8, 1, [(500, 2), (3, 1)], 130, 1),
    # pages in parts, of few rows and of many
    ("small", 64, 4, 2, [(1600, 2), (5, 1)], 0, 0),
    ("small", 64, 1, 1, [(760, 66)], 0, 0),
    ("small", 128, 2, 1, [(700, 40), (20, 33), (3, 1)], 0, 0),
    ("small", 64, 2, 1, [(1700, 3), (900, 50)], 800, 70),
    ("small", 64, 1, 1, [(860, 97)], 0, 0),
    ("small", 128, 3, 1, [(700, 40), (20, 33), (3, 1)], 0, 0),
    ("small", 64, 4, 1, [(1100, 30), (40, 25)], 900, 70),
    ("large", 64, 32, 8, [(300, 1)], 0, 0),
    ("large", 64, 32, 8, [(0, 1), (5000, 1), (64, 1), (1023, 1), (77, 1), (2048, 1)], 0, 0),
    ("large", 64, 32, 8, [(2000, 5), (100, 3), (0, 6), (700, 1)], 0, 0),
    ("large", 64, 32, 8, [(0, 333)], 0, 0),
    ("large", 64, 32, 8, [(517, 150), (900, 1), (64, 64)], 0, 0),
    ("large", 64, 32, 8, [(3000, 1), (10, 1), (1500, 40)], 512, 4),
    ("large", 64, 24, 3, [(130, 70), (900, 2)], 0, 0),
    ("large", 64, 40, 1, [(700, 9)], 0, 0),
    ("large", 128, 32, 8, [(1500, 6), (100, 2), (33, 1)], 0, 0),
    ("large", 128, 32, 4, [(200, 130)], 100, 130),
    ("large", 128, 16, 16, [(1000, 1), (0, 100)], 0, 0),
    ("large", 64, 4, 2, [(30000, 1)], 0, 0),
    ("large", 64, 4, 2, [(30000, 3)], 64, 2),
]


@pytest.mark.parametrize("size,dim,heads,kv_heads,seqs,window,sinks", SDPA)
def test_sdpa_paged(size, dim, heads, kv_heads, seqs, window, sinks):
    past, new = map(list, zip(*seqs))
    t = Step([a + b for a, b in seqs], kv_heads, dim, seed=heads + len(seqs))
    t.append([0] * len(seqs), past)
    plan = t.append(past, new)
    t.attend(plan, past, new, heads, window, sinks)


@pytest.mark.parametrize("rows", [1, 40, 60])
def test_sdpa_pages_of_very_different_size_small(rows):
    """Values (and keys) whose magnitude changes by page, up and down by up to
    2^100, with pages of zeros between: the sums' unit follows them."""
    n = 64 * 9
    t = Step([n + rows], 1, 64, half=0, seed=18 + rows)
    k, v = t.rows(n)
    size = np.array([1, 2.0**9, 2.0**-9, 0, 2.0**60, 2.0**-40, 2.0**-7, 2.0**7, 1], np.float32)
    v = v * np.repeat(size, 64)[:, None]
    k = k * np.repeat(np.array([1, 3, 1e-6, 1, 0, 1, 2, 1, 1], np.float32), 64)[:, None]
    for chosen in (size > 0, size < 2.0**50):  # the second: without the huge page
        keep = np.repeat(chosen, 64)
        t.append([0], [n], rows=(k, np.where(keep[:, None], v, 0)))
        plan = t.append([n], [rows])
        t.attend(plan, [n], [rows], 2)


@pytest.mark.parametrize("scale", [1e-3, 8.0])
def test_sdpa_flat_and_sharp_small(scale):
    """Nearly equal weights, and all of it on one position."""
    t = Step([150, 20], 2, 64, seed=11)
    t.append([0, 0], [149, 15])
    plan = t.append([149, 15], [1, 5])
    t.attend(plan, [149, 15], [1, 5], 4, scale=scale)


def test_sdpa_rotated_queries_small():
    t = Step([100], 2, 64, seed=12)
    plan = t.append([0], [100], rotated=True)
    t.attend(plan, [0], [100], 4, rotated=True)


def test_sdpa_zero_values_and_bad_queries_small():
    """Pages whose keys or values are all zero; a query that is not finite
    gives NaN in its own head's row and nowhere else."""
    t = Step([200], 2, 64, seed=13)
    k, v = t.rows(199)
    k[64:128], v[0:64] = 0, 0
    t.append([0], [199], rows=(k, v))
    plan = t.append([199], [1])
    t.attend(plan, [199], [1], 4)
    past, new, heads = [190], [10], 4
    plan = ops.KvPlan(t.pool, past, new, t.tables)
    q = t.r.standard_normal((10, heads * 64)).astype(np.float32)
    want, amp, vmax = S.sdpa(t.oracle[0], past, new, t.tables, q, heads)
    q[2, 70], q[9, 0] = np.inf, np.nan
    out = DeviceArray((10, heads * 64))
    ops.sdpa_paged(plan, 0, dev(q), out, heads)
    got = out.numpy().reshape(10, heads, 64)
    bad = np.zeros((10, heads), bool)
    bad[2, 1] = bad[9, 0] = True
    assert np.isnan(got[bad]).all() and not np.isnan(got[~bad]).any()
    got[bad] = want.reshape(got.shape)[bad]
    close(got.reshape(10, -1), want, amp, vmax, 64, 200)


def test_rows_do_not_depend_on_their_batch_small():
    """A sequence's rows alone and in a batch, at other pages: the same cache,
    and attention within the bound either way (checked against the oracle)."""
    t = Step([70, 90], 2, 64, seed=14)
    t.append([0, 0], [69, 80])
    plan = t.append([69, 80], [1, 10])
    t.attend(plan, [69, 80], [1, 10], 4)
    plan = ops.KvPlan(t.pool, [80], [10], t.tables[1:])
    q = t.r.standard_normal((10, 256)).astype(np.float32)
    out = DeviceArray((10, 256))
    ops.sdpa_paged(plan, 0, dev(q), out, 4)
    want, amp, vmax = S.sdpa(t.oracle[0], [80], [10], t.tables[1:], q, 4)
    close(out.numpy(), want, amp, vmax, 64, 90)


def test_sdpa_repeats_bit_for_bit():
    """No order of workgroups shows in the results."""
    t = Step([3000, 200, 41], 8, 64, seed=15)
    t.append([0, 0, 0], [2990, 199, 40])
    plan = t.append([2990, 199, 40], [10, 1, 1])
    q = dev(t.r.standard_normal((12, 32 * 64)).astype(np.float32))
    outs = []
    for _ in range(4):
        out = DeviceArray((12, 32 * 64))
        ops.sdpa_paged(plan, 0, q, out, 32)
        outs.append(out.numpy())
    assert all(np.array_equal(o, outs[0]) for o in outs)


def test_many_sequences_and_long_mixed_batch():
    """A decode batch of 700 sequences, and one with a long chat, a prompt and
    single tokens together (both kernels, cut and uncut pages)."""
    r = rng(30)
    past = list(r.integers(0, 130, 700))
    new = list(r.integers(0, 3, 700))
    t = Step([int(a + b) for a, b in zip(past, new)], 2, 64, seed=31)
    t.append([0] * 700, past)
    plan = t.append(past, new)
    t.check_cache(plan, past, new)
    t.attend(plan, past, new, 4)
    past, new = [20000, 40, 0, 700, 64], [1, 200, 1, 3, 64]
    t = Step([a + b for a, b in zip(past, new)], 2, 64, seed=32)
    t.append([0] * 5, past)
    plan = t.append(past, new)
    t.attend(plan, past, new, 8)
    t.attend(plan, past, new, 8, 1000, 5)


def test_pages_past_4_gib():
    """Pages whose bytes lie past 32 bits of offset."""
    n_pages = 600000  # 8 KB for each page and head
    pool = ops.KvPool(1, n_pages, 1, 64, S.inv_freq(32))
    r = rng(16)
    past, new = [100], [4]
    tables = np.array([[n_pages - 1, 555555]], np.uint32)
    small = S.Cache(2, 1, 64, S.inv_freq(32))
    at = np.array([[0, 1]], np.uint32)
    for a, b in (([0], past), (past, new)):
        k, v = r.standard_normal((2, b[0], 64)).astype(np.float32)
        plan = ops.KvPlan(pool, a, b, tables)
        ops.kv_append(plan, 0, dev(k), dev(v))
        small.append(a, b, at, k, v)
    k, v = DeviceArray((104, 1, 64)), DeviceArray((104, 1, 64))
    ops.kv_read(plan, 0, 104, k, v)
    assert np.array_equal(k.numpy(), small.values(at[0], 104, 0))
    assert np.array_equal(v.numpy(), small.values(at[0], 104, 1))
    q = r.standard_normal((4, 128)).astype(np.float32)
    out = DeviceArray((4, 128))
    ops.sdpa_paged(plan, 0, dev(q), out, 2)
    want, amp, vmax = S.sdpa(small, past, new, at, q, 2)
    close(out.numpy(), want, amp, vmax, 64, 104)


def test_two_threads_with_their_own_plans():
    """Calls of two threads over one pool, each its own sequences and plan."""
    t = Step([300, 500], 2, 64, seed=17)
    t.append([0, 0], [299, 450])
    plan = t.append([299, 450], [1, 50])
    parts = [([299], [1], t.tables[:1]), ([450], [50], t.tables[1:])]
    qs = [t.r.standard_normal((b[0], 256)).astype(np.float32) for _, b, _ in parts]
    errors = []

    def work(i):
        try:
            a, b, tab = parts[i]
            mine = ops.KvPlan(t.pool, a, b, tab)
            d_q, out = dev(qs[i]), DeviceArray(qs[i].shape)
            want, amp, vmax = S.sdpa(t.oracle[0], a, b, tab, qs[i], 4)
            for _ in range(20):
                ops.sdpa_paged(mine, 0, d_q, out, 4)
                close(out.numpy(), want, amp, vmax, 64, 500)
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert not errors, errors


# ---------------------------------------------------------------- refusals

def test_refusals_small():
    """Every refusal leaves the pool and the plan's former step as they were."""
    def code(f, *a, **kw):
        with pytest.raises((LLMError, KernelError)) as e:
            f(*a, **kw)
        return e.value.code

    inv = S.inv_freq(32)
    assert code(ops.KvPool, 1, 4, 2, 96, inv) == SQ_ERR_UNSUPPORTED
    assert code(ops.KvPool, 1, 4, 0, 64, inv) == SQ_ERR_SHAPE
    assert code(ops.KvPool, 1, 0, 2, 64, inv) == SQ_ERR_SHAPE
    assert code(ops.KvPool, 0, 4, 2, 64, inv) == SQ_ERR_SHAPE
    assert code(ops.KvPool, 1, 4, 2, 64, S.inv_freq(33)) == SQ_ERR_SHAPE
    assert code(ops.KvPool, 1, 4, 2, 64, np.array([np.nan], np.float32)) == SQ_ERR_ARG
    assert code(ops.KvPool, 1 << 30, 1 << 30, 4096, 128, inv) == SQ_ERR_SHAPE
    t = Step([70, 70], 2, 64, seed=20, spare=0)
    plan = t.append([0, 0], [70, 70])
    n_pages = 4
    bad = t.tables.copy()
    bad[1, 1] = n_pages
    assert code(plan.set, [0, 0], [70, 70], bad) == SQ_ERR_ARG  # past the pool
    bad[1, 1] = t.tables[0, 1]
    assert code(plan.set, [64, 64], [1, 1], bad) == SQ_ERR_ARG  # one page, two writers
    assert code(plan.set, [64, 65], [1, 0], bad) == SQ_ERR_ARG  # written and read
    bad[1] = t.tables[0]
    plan2 = ops.KvPlan(t.pool, [70, 70], [0, 0], bad)  # only read: shared pages are fine
    t.oracle[0].values(bad[0], 70, 0)
    assert code(plan.set, [0, 0], [70, 129], t.tables) == SQ_ERR_SHAPE  # table too short
    assert code(plan.set, [0, 0], [-1, 1], t.tables) == SQ_ERR_SHAPE
    assert code(plan.set, [0, 0], [70], t.tables) == SQ_ERR_SHAPE
    assert code(plan.set, [2**31 - 1, 0], [1, 0], t.tables) == SQ_ERR_SHAPE
    del plan2
    t.check_cache(plan, [0, 0], [70, 70])  # the former step
    k = DeviceArray((140, 128))
    small = DeviceArray((139, 128))
    assert code(ops.kv_append, plan, 0, small, k) == SQ_ERR_SHAPE
    assert code(ops.kv_append, plan, 1, k, k) == SQ_ERR_SHAPE  # no such layer
    assert code(ops.kv_append, plan, 0, k, k, k_stride=127) == SQ_ERR_SHAPE
    assert code(ops.sdpa_paged, plan, 0, k, k, 3) == SQ_ERR_SHAPE  # 3 heads, 2 KV heads
    assert code(ops.sdpa_paged, plan, 0, k, small, 2) == SQ_ERR_SHAPE
    assert code(ops.sdpa_paged, plan, 0, k, k, 0) == SQ_ERR_SHAPE
    assert code(ops.kv_read, plan, 0, 70, small, k) == SQ_ERR_SHAPE
    L = lib()
    assert L.sq_kv_append(None, 0, k.ptr, 128, k.ptr, 128, 0) == SQ_ERR_ARG
    assert L.sq_kv_append(plan.h, 0, None, 128, k.ptr, 128, 0) == SQ_ERR_ARG
    assert L.sq_kv_append(plan.h, 0, k.ptr, 128, k.ptr, 128, 2) == SQ_ERR_ARG
    assert L.sq_sdpa_paged(plan.h, 0, None, 128, k.ptr, 128, 2, 0, 0, 0) == SQ_ERR_ARG
    assert L.sq_sdpa_paged(plan.h, 0, k.ptr, 128, k.ptr, 128, 2, 0, 0, 4) == SQ_ERR_ARG
    assert L.sq_kv_read(plan.h, 0, 1, None, None) == SQ_ERR_ARG
    assert L.sq_kv_plan_set(plan.h, 1, None, None, None, 0) == SQ_ERR_ARG
    assert L.sq_kv_plan_set(plan.h, 65536, k.ptr, k.ptr, k.ptr, 0) == SQ_ERR_SHAPE  # refused before any is read
    t.check_cache(plan, [0, 0], [70, 70])


def test_read_sizes_small():
    """What kv_read gives for any `last`, and its refusals."""
    past, new = [3, 0, 100], [1, 0, 30]
    t = Step([4, 1, 130], 1, 64, seed=22)
    t.append([0, 0, 0], past)
    plan = t.append(past, new)
    for last in (0, 1, 4, 5, 129, 130, 1 << 40):
        assert plan.cached_rows(last) == sum(min(a + b, last) for a, b in zip(past, new))
        t.check_cache(plan, past, new, last=last)
    for last in (-1, 3):
        with pytest.raises(KernelError):
            ops.kv_read(plan, 0, last, DeviceArray((5, 64)), DeviceArray((5, 64)))


def test_steps_with_nothing_to_do_small():
    """No sequences, no rows, an unset plan: nothing runs, nothing is refused."""
    t = Step([10], 1, 64, seed=21)
    for plan in (ops.KvPlan(t.pool), ops.KvPlan(t.pool, [0], [0], t.tables),
                 ops.KvPlan(t.pool, [], [], np.zeros((0, 1), np.uint32))):
        none = DeviceArray((0, 64))
        ops.kv_append(plan, 0, none, none)
        ops.sdpa_paged(plan, 0, none, none, 1)
        ops.kv_read(plan, 0, 5, none, none)


# ---------------------------------------------------------------- verification

def drafts(r, n, vocab, temperature, near=0.7, sampled=True):
    n = np.asarray(n)
    rows = int(n.sum())
    target = (2.5 * r.standard_normal((rows + len(n), vocab))).astype(np.float32)
    of = np.concatenate([np.arange(k) + i + f for i, (f, k) in enumerate(zip(np.cumsum(n) - n, n))]).astype(int)
    draft = (target[of] + near * r.standard_normal((rows, vocab))).astype(np.float32)
    noise = -np.log(-np.log(r.uniform(1e-12, 1 - 1e-12, (rows, vocab))))
    tokens = (draft / max(temperature, 1e-3) + noise).argmax(1).astype(np.uint32) if rows else np.zeros(0, np.uint32)
    u = r.random(rows + len(n)).astype(np.float32)
    return target, draft if sampled else None, tokens, u


def run_verify(target, draft, tokens, u, n, temperature):
    got = ops.verify_draft(dev(target), None if draft is None else dev(draft), dev(tokens), dev(u), n, temperature)
    want = S.verify(target, draft, tokens, u, n, temperature)
    assert np.array_equal(got[0], want[0]), "accepted"
    assert np.array_equal(got[1], want[1]), "tokens"
    return got


VERIFY = [
    ("small", [1], 1, 1.0, True),
    ("small", [0], 7, 1.0, True),
    ("small", [3, 0, 1, 5], 257, 0.7, True),
    ("small", [2, 2], 4096, 1.3, True),
    ("small", [4], 4097, 1.0, False),
    ("small", [1, 3], 9000, 1.0, True),
    ("small", [3, 0, 2], 300, 0.0, True),
    ("large", [4], 128256, 0.8, True),
    ("large", [7, 0, 3, 1, 5, 2, 4, 7, 1, 0], 128256, 1.0, True),
    ("large", [3, 4, 5], 32001, 1.0, False),
    ("large", [3] * 40, 1000, 1.0, True),
    ("large", [2] * 300, 500, 0.9, True),
    ("large", [1, 0, 2] * 200, 300, 1.0, False),
    ("large", [40, 200], 700, 1.0, True),
    ("large", [5, 5], 128256, 0.0, False),
]


@pytest.mark.parametrize("size,n,vocab,temperature,sampled", VERIFY)
def test_verify_draft(size, n, vocab, temperature, sampled):
    r = rng(len(n) + vocab)
    target, draft, tokens, u = drafts(r, n, vocab, temperature, sampled=sampled)
    if temperature == 0.0 and len(tokens):  # some of the drafts right
        t0 = np.repeat(np.cumsum(np.asarray(n) + 1) - np.asarray(n) - 1, n) + np.arange(len(tokens)) - np.repeat(
            np.cumsum(n) - n, n)
        right = r.random(len(tokens)) < 0.8
        tokens[right] = target[t0].argmax(1)[right]
    run_verify(target, draft, tokens, u, n, temperature)


def test_verify_edges_small():
    r = rng(40)
    n, vocab = [3, 2, 2], 600
    target, draft, tokens, u = drafts(r, n, vocab, 1.0)
    for value in (0.0, np.float32(1 - 2.0**-24)):
        run_verify(target, draft, tokens, np.full_like(u, value), n, 1.0)
    # the draft is the target: everything is accepted
    same = target[[0, 1, 2, 4, 5, 7, 8]]
    acc, _ = run_verify(target, same, tokens, u * np.float32(0.999), n, 1.0)
    assert list(acc) == n
    # masked logits, the drafted token's among them, and all but one masked
    t2, d2 = target.copy(), draft.copy()
    t2[r.random(t2.shape) < 0.5] = -np.inf
    d2[r.random(d2.shape) < 0.3] = -np.inf
    t2[np.arange(10), np.arange(10)] = 1.0
    t2[6, np.arange(vocab) != 77] = -np.inf
    t2[6, 77] = -3.0
    run_verify(t2, d2, tokens, u, n, 1.0)
    run_verify(t2, None, tokens, u, n, 1.0)
    # neither has the drafted token and they agree elsewhere: drawn from p
    t3, d3 = target.copy(), same.copy()
    t3[0, tokens[0]] = d3[0, tokens[0]] = -np.inf
    acc, _ = run_verify(t3, d3, tokens, u, n, 1.0)
    assert acc[0] == 0
    # the weight at the first and at the last index, ties at temperature 0
    t4 = np.full((2, 5000), -np.inf, np.float32)
    t4[0, [0, 4999]], t4[1, [17, 4100]] = 0.0, 2.0
    for u0 in (0.1, 0.9):
        run_verify(t4, None, np.zeros(0, np.uint32), np.array([u0, 1 - u0], np.float32), [0, 0], 1.0)
    _, tok = run_verify(t4, None, np.zeros(0, np.uint32), np.zeros(2, np.float32), [0, 0], 0.0)
    assert list(tok) == [4999, 4100] and ops.greedy(dev(t4[0])) == 4999
    # logits and temperatures of any size
    for scale, temperature in ((1e30, 1.0), (1e-30, 1.0), (1.0, 1e-30), (1.0, 1e30)):
        run_verify((target * np.float32(scale)).astype(np.float32), (draft * np.float32(scale)).astype(np.float32),
                   tokens, u, n, temperature)


def test_verify_strided_rows_small():
    """Rows a few floats apart, at an address that is a multiple of 4 only."""
    r = rng(41)
    n, vocab = np.array([2, 1], np.uint32), 333
    target, draft, tokens, u = drafts(r, n, vocab, 1.0)
    t, d = np.full((5, 337), np.nan, np.float32), np.full((3, 334), np.nan, np.float32)
    t[:, 1:1 + vocab], d[:, 1:] = target, draft
    d_t, d_d, d_tok, d_u = dev(t), dev(d), dev(tokens), dev(u)
    acc, tok = np.zeros(2, np.uint32), np.zeros(2, np.uint32)
    assert lib().sq_verify_draft(d_t.ptr + 4, 337, d_d.ptr + 4, 334, d_tok.ptr, d_u.ptr, n.ctypes.data, 2, vocab, 1.0,
                                 acc.ctypes.data, tok.ctypes.data) == 0
    want = S.verify(target, draft, tokens, u, n, 1.0)
    assert np.array_equal(acc, want[0]) and np.array_equal(tok, want[1])


def test_verify_refusals_small():
    r = rng(42)
    n, vocab = np.array([2, 1], np.uint32), 5000
    target, draft, tokens, u = drafts(r, n, vocab, 1.0)

    def code(target=target, draft=draft, tokens=tokens, u=u, n=n, temperature=1.0):
        with pytest.raises((LLMError, KernelError)) as e:
            ops.verify_draft(dev(target), None if draft is None else dev(draft), dev(tokens), dev(u), n, temperature)
        return e.value.code

    u0 = np.zeros_like(u)  # every draft with p > 0 is accepted
    for value in (np.nan, np.inf):
        for at in (0, 4321):
            t = target.copy()
            t[1, at] = value
            assert code(target=t, u=u0) == SQ_ERR_ARG
            assert code(target=t, u=u0, temperature=0.0, tokens=target.argmax(1).astype(np.uint32)[[0, 1, 3]]) == SQ_ERR_ARG
            d = draft.copy()
            d[2, at] = value
            assert code(draft=d, u=u0) == SQ_ERR_ARG
    t = target.copy()
    t[3] = -np.inf
    assert code(target=t, u=u0) == SQ_ERR_ARG
    for bad in (vocab, 2**32 - 1):
        x = tokens.copy()
        x[2] = bad
        assert code(tokens=x) == SQ_ERR_ARG
    assert code(temperature=-1.0) == code(temperature=float("nan")) == code(temperature=float("inf")) == SQ_ERR_ARG
    assert code(n=[2, 2]) == SQ_ERR_SHAPE
    assert code(n=[1025, 0]) == SQ_ERR_SHAPE
    assert code(draft=draft[:, :-1]) == SQ_ERR_SHAPE
    acc = np.full(2, 99, np.uint32)
    d_t, d_tok, d_u = dev(target), dev(np.array([vocab, 0, 0], np.uint32)), dev(u)
    assert lib().sq_verify_draft(d_t.ptr, vocab, None, 0, d_tok.ptr, d_u.ptr, n.ctypes.data, 2, vocab, 1.0,
                                 acc.ctypes.data, acc.ctypes.data) == SQ_ERR_ARG
    assert list(acc) == [99, 99]  # left as they were
    assert lib().sq_verify_draft(d_t.ptr, vocab - 1, None, 0, d_tok.ptr, d_u.ptr, n.ctypes.data, 2, vocab, 1.0,
                                 acc.ctypes.data, acc.ctypes.data) == SQ_ERR_SHAPE
    assert lib().sq_verify_draft(None, vocab, None, 0, d_tok.ptr, d_u.ptr, n.ctypes.data, 2, vocab, 1.0,
                                 acc.ctypes.data, acc.ctypes.data) == SQ_ERR_ARG


def test_rows_behind_a_rejection_may_hold_anything_small():
    r = rng(43)
    n, vocab = [3, 1], 700
    target, draft, tokens, u = drafts(r, n, vocab, 1.0)
    target[0, tokens[0]] = -np.inf  # the first draft is rejected
    want = S.verify(target, draft, tokens, u, n, 1.0)
    target[1:4], draft[1:3] = np.nan, np.inf
    tokens[1] = vocab + 5
    got = ops.verify_draft(dev(target), dev(draft), dev(tokens), dev(u), n, 1.0)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("size,dim,window,sinks", [("small", 64, 0, 0), ("small", 64, 70, 3), ("large", 128, 0, 0),
                                                   ("large", 64, 300, 4)])
def test_serving_steps(size, dim, window, sinks):
    """Steps of a server with drafts: each layer's append and attention over the
    drafted rows, the verification of what the last layer's rows score, the
    rejected rows overwritten by the next step."""
    layers, kv_heads, heads = 2, 2, 4
    lens = [70, 5, 130] if size == "small" else [700, 5, 1300, 64]
    steps, vocab = (3, 300) if size == "small" else (6, 5000)
    t = Step([n + 8 * steps for n in lens], kv_heads, dim, layers=layers, seed=50)
    for layer in range(layers):
        t.append([0] * len(lens), lens, layer=layer)
    past = np.array(lens)
    head = t.r.standard_normal((heads * dim, vocab)).astype(np.float32) * np.float32(0.3)
    for step in range(steps):
        n = t.r.integers(0, 6, len(past))
        new = n + 1  # the last known token and its drafts
        for layer in range(layers):
            plan = t.append(past, new, layer=layer)
            t.attend(plan, past, new, heads, window, sinks, layer=layer)
        q = t.r.standard_normal((int(new.sum()), heads * dim)).astype(np.float32)
        out = DeviceArray(q.shape)
        ops.sdpa_paged(plan, layers - 1, dev(q), out, heads, window=window, sinks=sinks)
        target = (out.numpy() @ head).astype(np.float32)
        _, draft, tokens, u = drafts(t.r, n, vocab, 1.0)
        acc, _ = run_verify(target, draft, tokens, u, n, 1.0)
        past = past + 1 + acc
    t.check_cache(plan, past - 1 - acc, new, layer=layers - 1)
