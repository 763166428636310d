"""The paged KV cache on the device (ort_cuda_paged_kv_append,
ort_cuda_paged_attention) against the float64 formulas of
tests/paged_reference.py.

Tolerances.  Attention: the exact mode's bar, max|dY| / max|Y_ref| <= 1e-5
(fp32 products and sums: a score of D = 128 products is off by about
sqrt(128) * 2^-24 * |s|, a weight by as much relative to itself, and the
weighted sum averages these).  fp32 cache rows and rotated queries are the
double result rounded once: equal.  16-bit cache rows: half a step of the
type, 2^-11 (fp16) or 2^-8 (bf16) of the value.
"""
import math

import pytest
import torch

from tests import paged_reference as ref
from tests.conftest import max_rel

pytestmark = pytest.mark.gpu
TOL = 1e-5
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def sess():
    from onnx_runtime_dart_b200 import CudaSession
    s = CudaSession(0)
    yield s
    s.close()


def handle(s):
    from onnx_runtime_dart_b200 import PagedKVCache
    return PagedKVCache(s["key"], s["value"], s["table"], s["cu"], s["past"])


def run(sess, s, heads, new, checked=True, **kw):
    kw.setdefault("max_seq", max(new + [0]))
    out = sess.paged_attention(handle(s), s["q"], heads, **kw)
    if checked:
        sess.sync()  # raises what a kernel reported: a wait that ran out, lengths that do not fit
    return out


def near(want, got, tol=TOL):
    assert torch.isfinite(got).all()
    err = max_rel(want.cpu().numpy(), got.double().cpu().numpy())
    assert err <= tol, err


# new lengths, past lengths, heads, kv heads, head, page
SHAPES = [
    ([1], [0], 4, 4, 64, 16),                        # one key: its own
    ([1], [639], 32, 8, 64, 16),
    ([1], [5000], 8, 1, 128, 16),                    # a long axis, few rows
    ([1] * 9, [0, 1, 15, 16, 17, 127, 128, 129, 1000], 32, 8, 128, 16),
    ([1, 0, 1], [300, 40, 0], 16, 2, 128, 64),       # a sequence without tokens
    ([3, 1, 8, 5], [70, 0, 33, 900], 16, 8, 64, 24),  # drafted tokens, pages of 24
    ([2, 9], [3, 200], 12, 12, 80, 7),               # odd pages, head 80, one head a group
    ([17], [0], 8, 2, 8, 5),
    ([1, 40], [100, 3], 40, 8, 96, 33),
    ([130], [0], 32, 8, 128, 16),
    ([300, 1, 65], [0, 700, 129], 8, 2, 64, 256),
    ([257, 255], [511, 0], 16, 4, 128, 16),
    ([500], [77], 7, 1, 120, 40),                    # seven heads a group
    ([33], [20], 64, 1, 32, 16),                     # sixty-four heads a group
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(sess, shape, dtype):
    new, past, heads, kv_heads, head, page = shape
    s = ref.make(1, dtype, new, past, heads, kv_heads, head, page)
    want = ref.attention(s, new, past, heads)
    got = run(sess, s, heads, new)
    near(want, got)
    again = run(sess, s, heads, new, max_seq=None)  # a looser bound of the lengths
    near(want, again)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("window,softcap,scale", [(1, 0.0, None), (50, 0.0, None),
                                                  (0, 5.0, 0.3), (200, 30.0, None),
                                                  (100000, 0.0, 0.01)])
@pytest.mark.parametrize("shape", [([1, 1, 2], [40, 900, 10], 16, 4, 128, 16),
                                   ([150, 300], [60, 0], 8, 2, 64, 16)])
def test_attention_window_softcap_scale(sess, shape, window, softcap, scale, dtype):
    new, past, heads, kv_heads, head, page = shape
    s = ref.make(2, dtype, new, past, heads, kv_heads, head, page)
    want = ref.attention(s, new, past, heads, scale, softcap, window)
    near(want, run(sess, s, heads, new, scale=scale, softcap=softcap,
                   local_window_size=window))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (120, 20.0), (1000, 0.0)])
@pytest.mark.parametrize("shared,shape", [
    (128, ([1] * 5, [128, 130, 200, 128, 400], 32, 8, 128, 16)),
    (1000, ([1] * 20, [1000 + 7 * i for i in range(20)], 32, 8, 128, 16)),
    (500, ([2, 0, 1, 3], [500, 0, 640, 501], 16, 8, 64, 64)),      # ends inside a page
    (1, ([1, 1], [1, 90], 8, 8, 64, 16)),
    (333, ([70, 1, 40], [333, 500, 350], 8, 2, 64, 16)),           # prompts behind it
    (700, ([1] * 70, [701 + i for i in range(70)], 8, 1, 96, 32)),
])
def test_attention_shared_prefix(sess, shared, shape, window, softcap, dtype):
    new, past, heads, kv_heads, head, page = shape
    s = ref.make(3, dtype, new, past, heads, kv_heads, head, page, shared)
    want = ref.attention(s, new, past, heads, None, softcap, window)
    near(want, run(sess, s, heads, new, softcap=softcap, local_window_size=window,
                   shared_len=shared))
    near(want, run(sess, s, heads, new, softcap=softcap, local_window_size=window))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,past", [([1], 900), ([1, 0, 2], 70), ([40], 30), ([1, 33, 1], 200)])
def test_attention_many_sequences(sess, new, past, dtype):
    """More sequences than a block has threads: the list is found in two passes."""
    batch = 700
    new = [new[b % len(new)] for b in range(batch)]
    past = [(b * 37) % past for b in range(batch)]
    s = ref.make(16, dtype, new, past, 8, 2, 64, 16)
    want = ref.attention(s, new, past, 8)
    near(want, run(sess, s, 8, new))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("window", [0, 700])
def test_attention_long_prompt(sess, window, dtype):
    """Many tiles of rows per run, long and short ones, on every kind of page."""
    for page in (16, 12):
        new, past = [2600, 500], [0, 1300]
        s = ref.make(17, dtype, new, past, 8, 2, 128, page)
        want = ref.attention(s, new, past, 8, window=window)
        near(want, run(sess, s, 8, new, local_window_size=window))


def test_attention_of_drawn_batches(sess):
    """Ragged batches of all kinds, drawn from a seed."""
    import random
    for seed in range(40):
        r = random.Random(seed)
        heads, G = r.choice([(8, 8), (8, 2), (16, 1), (12, 4), (7, 1), (32, 8)])
        head, page = r.choice([64, 128, 96, 72]), r.choice([16, 8, 64, 24, 11, 1, 48])
        batch = r.choice([1, 2, 5, 17, 60])
        most = r.choice([1, 1, 4, 30, 200])
        new = [r.randint(0, most) for _ in range(batch)]
        new[r.randrange(batch)] = most
        shared = r.choice([0, 0, r.randint(1, 500)])
        past = [shared + int(10 ** r.uniform(0, 3.3)) for _ in range(batch)]
        window = r.choice([0, 0, r.randint(1, 600)])
        softcap = r.choice([0.0, 0.0, 10.0])
        s = ref.make(seed, r.choice([F32, F16, BF16]), new, past, heads, G, head, page, shared)
        want = ref.attention(s, new, past, heads, None, softcap, window)
        near(want, run(sess, s, heads, new, softcap=softcap, local_window_size=window,
                       shared_len=shared))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_large_and_small_values(sess, dtype):
    """Queries over ten orders of magnitude, sharp and flat rows."""
    new, past, heads = [6, 140], [90, 0], 8
    s = ref.make(4, dtype, new, past, heads, 2, 64, 16)
    s["q"] *= torch.logspace(-6, 1.0, sum(new), device="cuda")[:, None]
    want = ref.attention(s, new, past, heads)
    near(want, run(sess, s, heads, new))


def test_q_rows_apart_and_three_dimensions(sess):
    """Queries that are a slice of a fused projection's output."""
    new, past, heads, G, D = [1, 4, 150], [30, 5, 2], 8, 2, 64
    s = ref.make(5, F16, new, past, heads, G, D, 16)
    fused = torch.randn((sum(new), (heads + 2 * G) * D + 3), device="cuda")
    fused[:, 1:1 + heads * D] = s["q"]
    want = ref.attention(s, new, past, heads)
    s["q"] = fused[:, 1:1 + heads * D]
    near(want, run(sess, s, heads, new))
    s["q"] = s["q"].unflatten(1, (heads, D))
    got = run(sess, s, heads, new)
    assert got.shape == (sum(new), heads, D)
    near(want, got.flatten(1))
    near(want, run(sess, {**s, "q": s["q"].double()}, heads, new).flatten(1))


def test_padding_rows_are_left(sess):
    """Tokens behind the last sequence: their output rows, and the cache, stay."""
    new, past, heads, G, D = [1, 3, 0, 200], [9, 0, 4, 30], 8, 4, 64
    s = ref.make(6, F16, new, past, heads, G, D, 16)
    pad = 37
    q = torch.cat([s["q"], torch.full((pad, heads * D), math.nan, device="cuda")])
    out = torch.full_like(q, 7.0)
    got = run(sess, {**s, "q": q}, heads, new, out=out)
    assert got is out
    near(ref.attention(s, new, past, heads), got[:sum(new)])
    assert (got[sum(new):] == 7.0).all()
    before = s["key"].clone(), s["value"].clone()
    kv = torch.full((pad, G * D), 3.0, device="cuda")
    s["cu"].zero_()
    sess.paged_kv_append(handle(s), kv, kv)
    assert torch.equal(before[0].view(torch.int16), s["key"].view(torch.int16))
    assert torch.equal(before[1].view(torch.int16), s["value"].view(torch.int16))


def test_no_tokens(sess):
    s = ref.make(7, F16, [1], [3], 4, 4, 64, 16)
    empty = torch.empty((0, 256), device="cuda")
    assert sess.paged_attention(handle(s), empty, 4).shape == (0, 256)
    assert sess.paged_kv_append(handle(s), empty, empty) is None
    none = {**s, "table": s["table"][:0], "cu": s["cu"][:1], "past": s["past"][:0]}
    out = torch.full((2, 256), 5.0, device="cuda")
    sess.paged_attention(handle(none), torch.zeros((2, 256), device="cuda"), 4, out=out)
    assert (out == 5.0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,past,window", [([4, 40], [20, 60], 0), ([3], [200], 30),
                                             ([200], [50], 0), ([140, 170], [300, 0], 64)])
def test_infinite_and_nan_values_in_masked_places(sess, new, past, window, dtype):
    """A key or value that a row does not see has no part in it, whatever it
    holds: later tokens of the same prompt, keys before the window."""
    heads, G, D = 8, 2, 64
    s = ref.make(8, dtype, new, past, heads, G, D, 16)
    clean = {k: v.clone() for k, v in s.items()}
    rows = torch.zeros(sum(new), dtype=torch.bool)  # rows that see a planted key
    row = 0
    for b, (n, p0) in enumerate(zip(new, past)):
        plants = [(p0 + n - 2, math.inf), (p0 + n - 1, math.nan)]
        if window and p0 >= window:
            plants.append((p0 - window, -math.inf))
        for j, x in plants:
            page, at = int(s["table"][b, j // 16]), j % 16
            s["value"][page, at, :, 3::7] = x
            s["key"][page, at, :, 5::9] = x
            for i in range(n):
                if j <= p0 + i and (not window or j > p0 + i - window):
                    rows[row + i] = True
        row += n
    want = ref.attention(clean, new, past, heads, None, 0.0, window)
    got = run(sess, s, heads, new, local_window_size=window)
    assert not torch.isfinite(got[rows.cuda()]).all()
    near(want[~rows.cuda()], got[~rows.cuda()])


def test_pages_behind_2_31_elements(sess):
    """Pages whose offset in elements and bytes passes 32 bits."""
    new, past, heads, G, D = [1, 130], [500, 10], 16, 8, 128
    s = ref.make(9, F16, new, past, heads, G, D, 16)
    want = ref.attention(s, new, past, heads)
    count = (1 << 31) // (16 * G * D) + 100
    big = {**s}
    for name in ("key", "value"):
        big[name] = torch.empty((count, 16, G, D), dtype=F16, device="cuda")
        big[name][-s[name].shape[0]:] = s[name]
    big["table"] = torch.where(s["table"] < 0, -1, s["table"] + count - s["key"].shape[0]).int()
    near(want, run(sess, big, heads, new))
    k = torch.randn((sum(new), G * D), device="cuda")
    sess.paged_kv_append(handle(big), k, k)
    page = int(big["table"][0, 500 // 16])
    assert torch.equal(big["key"][page, 500 % 16].flatten(), k[0].half())
    del big


# ---- append ---------------------------------------------------------------------

def half_step(dtype):
    return 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape,half", [
    (([1], [0], 4, 4, 64, 16), 32),
    (([1] * 5, [0, 15, 16, 300, 1], 32, 8, 128, 16), 64),
    (([40, 0, 3], [2, 9, 100], 12, 12, 80, 7), 40),
    (([5, 300], [31, 0], 8, 1, 96, 33), 24),      # a part of the head is rotated
    (([2], [3], 2, 1, 8, 1), 3),
    (([9, 1], [4, 60], 8, 2, 128, 24), 0),         # no rotation
])
def test_append(sess, shape, half, interleaved, dtype):
    new, past, heads, G, D, page = shape
    s = ref.make(10, dtype, new, past, heads, G, D, page)
    n = sum(new)
    g = torch.Generator().manual_seed(11)
    k, v = (torch.randn((n, G * D), generator=g).cuda() for _ in range(2))
    pos = torch.cat([torch.arange(p0, p0 + m) for m, p0 in zip(new, past)]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    kw, q_want, k_want = {}, s["q"].double(), k.view(n, G, D).double()
    if half:
        ang = torch.rand((int(pos.max()) + 2, half), generator=g, dtype=torch.float64).cuda() * 6.3
        cos, sin = ang.cos().float(), ang.sin().float()
        kw = dict(cos_cache=cos, sin_cache=sin, rotary_interleaved=interleaved)
        q_want = ref.rotate(s["q"].view(n, heads, D), cos[pos], sin[pos], interleaved).view(n, -1)
        k_want = ref.rotate(k_want, cos[pos], sin[pos], interleaved)
    where = (s["table"][seq, pos // page].long(), pos % page)
    key, value = s["key"].clone(), s["value"].clone()
    got = sess.paged_kv_append(handle(s), k, v, q=s["q"], num_heads=heads, **kw)
    assert torch.equal(got, q_want.float())
    step = half_step(dtype)
    for cache, want in ((s["key"], k_want), (s["value"], v.view(n, G, D).double())):
        have = cache[where].double()
        if dtype == F32:
            assert torch.equal(have, want.float().double())
        assert ((have - want).abs() <= step * (1 + 1e-6) * want.abs() + 2.0 ** -25).all() or \
            dtype == F32
    # every other row is as it was (bit for bit, NaN rows among them)
    key[where], value[where] = s["key"][where], s["value"][where]
    word = torch.int32 if dtype == F32 else torch.int16
    assert torch.equal(key.view(word), s["key"].view(word))
    assert torch.equal(value.view(word), s["value"].view(word))
    # in place, and without queries
    q = s["q"].clone()
    assert sess.paged_kv_append(handle(s), k, v, q=q, num_heads=heads, q_out=q, **kw) is q
    assert torch.equal(q, got)
    assert sess.paged_kv_append(handle(s), k, v, **kw) is None


def test_append_rows_apart(sess):
    """k, v and q as slices of one fused projection, at an odd offset too."""
    new, past, heads, G, D = [3, 1], [10, 50], 8, 2, 64
    for lead in (0, 1):
        s = ref.make(12, F16, new, past, heads, G, D, 16)
        fused = torch.randn((4, lead + (heads + 2 * G) * D), device="cuda")
        q, k, v = fused[:, lead:].split([heads * D, G * D, G * D], dim=1)
        ang = torch.rand((60, D // 2), device="cuda") * 6.3
        kw = dict(num_heads=heads, cos_cache=ang.cos(), sin_cache=ang.sin())
        t = {n: x.clone() for n, x in s.items()}
        a = sess.paged_kv_append(handle(s), k, v, q=q, **kw)
        b = sess.paged_kv_append(handle(t), k.contiguous(), v.contiguous(), q=q.contiguous(), **kw)
        assert torch.equal(a, b)
        assert torch.equal(s["key"].view(torch.int16), t["key"].view(torch.int16))
        assert torch.equal(s["value"].view(torch.int16), t["value"].view(torch.int16))


# ---- what does not fit --------------------------------------------------------------

def reported(sess, text):
    with pytest.raises(ValueError, match=text):
        sess.sync()
    sess.sync()


@pytest.mark.parametrize("new", [[1, 2, 1], [70, 130, 90]])
def test_bad_pages_and_lengths_are_left_out(sess, new):
    past, heads, G, D = [40, 60, 20], 8, 2, 64
    s = ref.make(13, F16, new, past, heads, G, D, 16)
    want = ref.attention(s, new, past, heads)
    kv = torch.zeros((sum(new), G * D), device="cuda")
    first, last = slice(0, new[0]), slice(new[0] + new[1], None)
    for bad in (-5, s["key"].shape[0], 2 ** 31 - 1):  # keys of one page of sequence 1
        t = {**s, "table": s["table"].clone()}
        t["table"][1, 1] = bad
        got = run(sess, t, heads, new, checked=False)
        near(want[first], got[first])
        near(want[last], got[last])
        reported(sess, "page")
    t["table"][1, past[1] // 16] = -1
    sess.paged_kv_append(handle({**t, "key": s["key"].clone(), "value": s["value"].clone()}),
                         kv, kv)
    reported(sess, "page")
    for name, at, x in (("past", 1, -1), ("past", 1, 16 * s["table"].shape[1] - new[1] + 1),
                        ("past", 1, 2 ** 31 - 1), ("cu", 2, 0)):
        t = {**s, name: s[name].clone()}
        t[name][at] = x
        out = torch.full_like(s["q"], 7.0)
        run(sess, t, heads, new, checked=False, out=out)
        near(want[first], out[first])
        assert (out[new[0]:new[0] + new[1]] == 7.0).all() or name == "cu"
        reported(sess, "cu_seqlens")
        sess.paged_kv_append(handle({**t, "key": s["key"].clone(), "value": s["value"].clone()}),
                             kv, kv)
        reported(sess, "cu_seqlens")
    # more tokens than max_seq, than num_tokens, a past shorter than the shared prefix
    out = torch.full_like(s["q"], 7.0)
    run(sess, s, heads, new, checked=False, out=out, max_seq=max(new) - 1)
    assert (out[new[0]:new[0] + new[1]] == 7.0).all()
    near(want[first], out[first])
    reported(sess, "max_seq")
    out = torch.full_like(s["q"][:-1], 7.0)
    run(sess, {**s, "q": s["q"][:-1]}, heads, new, checked=False, out=out)
    assert (out[last] == 7.0).all()
    near(want[first], out[first])
    reported(sess, "num_tokens")
    t = {**s, "past": s["past"].clone()}
    t["past"][2] = 15
    out = torch.full_like(s["q"], 7.0)
    run(sess, t, heads, new, checked=False, out=out, shared_len=16)
    assert (out[last] == 7.0).all()
    reported(sess, "shared_len")
    near(want, run(sess, s, heads, new))


def test_position_outside_the_caches_is_left_out(sess):
    s = ref.make(14, F32, [1, 1], [3, 9], 4, 4, 64, 16)
    k = torch.randn((2, 256), device="cuda")
    cos = torch.ones((5, 32), device="cuda")
    key = s["key"].clone()
    sess.paged_kv_append(handle(s), k, k, cos_cache=cos, sin_cache=cos * 0)
    reported(sess, "position")
    page = int(s["table"][1, 0])
    assert torch.equal(s["key"][page, 9].isnan(), key[page, 9].isnan())
    assert torch.equal(s["key"][int(s["table"][0, 0]), 3].flatten(), k[0])


def test_refusals(sess):
    from onnx_runtime_dart_b200 import PagedKVCache, UnsupportedError
    s = ref.make(15, F16, [2], [5], 8, 2, 64, 16)
    h, q = handle(s), s["q"]
    kv = torch.zeros((2, 128), device="cuda")
    for call in (lambda: sess.paged_attention(h, q, 7),
                 lambda: sess.paged_attention(h, q[:, :-64], 7),
                 lambda: sess.paged_attention(h, q.cpu(), 8),
                 lambda: sess.paged_attention(h, q.int(), 8),
                 lambda: sess.paged_attention(h, q, 8, max_seq=-1),
                 lambda: sess.paged_attention(h, q, 8, shared_len=-1),
                 lambda: sess.paged_attention(h, q, 8, shared_len=10 ** 6),
                 lambda: sess.paged_attention(h, q, 8, scale=math.inf),
                 lambda: sess.paged_attention(h, q, 8, softcap=math.nan),
                 lambda: sess.paged_attention(h, q, 8, out=q),
                 lambda: sess.paged_attention(h, q.cpu().numpy(), 8),
                 lambda: sess.paged_kv_append(h, None, kv),
                 lambda: sess.dispatch(
                     dict(op_type="PagedAttention", inputs=list("q__kvcpb"),
                          attrs=dict(num_heads=8, kv_num_heads=2)),
                     dict(zip("q_kvcpb", [q.cpu().numpy(), None, s["key"], s["value"], s["cu"],
                                          s["past"], s["table"]]))),
                 lambda: sess.paged_kv_append(h, q[:, :128].contiguous(), kv, q=q, num_heads=8,
                                              q_out=torch.empty(2, 513, device="cuda")[:, 1:]),
                 lambda: sess.paged_attention(h, q, 8, out=q.half()),
                 lambda: sess.paged_attention(h, q, 8, out=q[:1]),
                 lambda: sess.paged_kv_append(h, kv, kv[:1]),
                 lambda: sess.paged_kv_append(h, kv[:, :64], kv),
                 lambda: sess.paged_kv_append(h, kv, kv, q=q, num_heads=3),
                 lambda: sess.paged_kv_append(h, kv, kv, q_out=q),
                 lambda: sess.paged_kv_append(h, kv, kv, cos_cache=kv),
                 lambda: sess.paged_kv_append(h, kv, kv, cos_cache=kv, sin_cache=kv),
                 lambda: sess.dispatch(
                     dict(op_type="PagedAttention", inputs=list("qxykvcpb"),
                          attrs=dict(num_heads=8, kv_num_heads=2, do_rotary=1)),
                     dict(q=q, x=kv, y=kv, k=s["key"], v=s["value"], c=s["cu"], p=s["past"],
                          b=s["table"])),
                 lambda: PagedKVCache(s["key"], s["value"].float(), s["table"], s["cu"], s["past"]),
                 lambda: PagedKVCache(s["key"], s["value"], s["table"].long(), s["cu"], s["past"]),
                 lambda: PagedKVCache(s["key"], s["value"], s["table"], s["cu"][:1], s["past"]),
                 lambda: PagedKVCache(s["key"].transpose(1, 2), s["value"], s["table"], s["cu"],
                                      s["past"]),
                 lambda: PagedKVCache(s["key"].cpu(), s["value"], s["table"], s["cu"], s["past"])):
        with pytest.raises(ValueError):
            call()
    both = torch.zeros((3, 512), device="cuda")
    with pytest.raises(ValueError, match="overlap"):  # shifted by a row
        sess.paged_kv_append(h, kv, kv, q=both[:2], num_heads=8, q_out=both[1:])
    with pytest.raises(ValueError, match="overlaps K"):
        sess.paged_kv_append(h, both[0, :256].view(2, 128), kv, q=q, num_heads=8, q_out=both[:2])
    for head in (136, 12):
        odd = ref.make(15, F16, [2], [5], 2, 1, head, 16)
        with pytest.raises(UnsupportedError):
            sess.paged_attention(handle(odd), odd["q"], 2)
    with pytest.raises(UnsupportedError):
        PagedKVCache(s["key"].double(), s["value"].double(), s["table"], s["cu"], s["past"])
    from onnx_runtime_dart_b200 import _lib
    L = _lib.load()
    assert L.ort_cuda_paged_attention(sess.handle, h.ref, q.data_ptr(), 512, 2, 2, 8, 0.0, 0.0,
                                      -1, 0, 0, 0) == _lib.ERR_INVALID_ARG
    assert L.ort_cuda_paged_attention(sess.handle, h.ref, q.data_ptr(), 512, 2, 2, 8, 0.0, 0.0,
                                      -1, 0, q.data_ptr(), _lib.HOST_IO) == _lib.ERR_INVALID_ARG


# ---- streams, graphs, the whole step ---------------------------------------------------

def test_two_streams_at_once(sess):
    """Calls of one session on two streams overlap without sharing a workspace."""
    cases = []
    for i, (new, past) in enumerate((([1] * 8, [4000] * 8), ([1] * 3, [9000] * 3),
                                     ([300, 200], [0, 900]))):
        s = ref.make(20 + i, F16, new, past, 8, 2, 128, 16)
        cases.append((s, new, run(sess, s, 8, new).clone()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[] for _ in cases]
    for _ in range(20):
        for (s, new, _), st, o in zip(cases, streams, outs):
            with torch.cuda.stream(st):
                o.append(run(sess, s, 8, new, checked=False))
    torch.cuda.synchronize()
    sess.sync()
    for (_, _, want), o in zip(cases, outs):
        for got in o:
            assert torch.equal(want, got)


def test_explicit_stream(sess):
    s = ref.make(23, F16, [1, 5], [700, 3], 8, 2, 64, 16)
    want = run(sess, s, 8, [1, 5])
    s["q"] = s["q"].double()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    sess.set_stream(st.cuda_stream)
    try:
        got = run(sess, s, 8, [1, 5])
        st.synchronize()
        assert torch.equal(want, got)
    finally:
        sess.set_stream(None)


@pytest.mark.parametrize("new", [[1, 1, 1], [90, 1, 140]])
def test_captured_call_follows_lengths_and_graphs_run_at_once(sess, new):
    """A captured append and attention replayed with new lengths and pages, and
    two captured graphs replayed at the same time."""
    past, heads, G, D = [3000, 40, 1500], 8, 2, 64
    room = [p + 64 for p in past]
    graphs = []
    for seed in (24, 25):
        s = ref.make(seed, F16, new, room, heads, G, D, 16, garbage=False)
        s["past"].copy_(torch.tensor(past))
        k, v = (torch.randn((sum(new), G * D), device="cuda") for _ in range(2))
        q, out, h = s["q"].clone(), torch.zeros_like(s["q"]), handle(s)
        ang = torch.rand((max(room) + max(new), D // 2), device="cuda") * 6.3
        cos, sin = ang.cos(), ang.sin()

        def step(s=s, k=k, v=v, q=q, out=out, h=h, cos=cos, sin=sin):
            sess.paged_kv_append(h, k, v, q=s["q"], num_heads=heads, cos_cache=cos, sin_cache=sin,
                                 q_out=q)
            sess.paged_attention(h, q, heads, max_seq=max(new), out=out)

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):  # nothing was run before: workspaces come with the graph
            step()
        graphs.append((graph, s, step, out))
    for add in (0, 1, 50):
        wants = []
        for _, s, step, out in graphs:
            s["past"].copy_(torch.tensor([p + add for p in past]))
            step()
            wants.append(out.clone())
            out.zero_()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(5):
            for (graph, *_), st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, out), want in zip(graphs, wants):
            assert torch.equal(out, want)
    sess.sync()


def test_session_graph(sess):
    """The session's own recording (ort_cuda_graph_begin) with an explicit stream."""
    s = ref.make(26, F16, [1, 1], [900, 20], 8, 2, 64, 16)
    want = run(sess, s, 8, [1, 1])
    out, h = torch.zeros_like(s["q"]), handle(s)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    sess.set_stream(st.cuda_stream)
    try:
        sess.graph_begin()
        sess.paged_attention(h, s["q"], 8, max_seq=1, out=out)
        gid = sess.graph_end()
        for _ in range(3):
            out.zero_()
            torch.cuda.synchronize()
            sess.graph_launch(gid)
            sess.sync()
            assert torch.equal(out, want)
        sess.graph_drop(gid)
    finally:
        sess.set_stream(None)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("packed", [False, True])
def test_dispatch_steps_match_dense_attention(sess, dtype, packed):
    """A prompt and six steps through dispatch('PagedAttention'), beside
    GroupQueryAttention with a dense cache of the same sequence (fp32 pages),
    or the float64 formula over the pages."""
    from onnx_runtime_dart_b200 import PagedKVCache
    heads, G, D, page, room = 8, 2, 64, 16, 96
    table = torch.randperm(12, generator=torch.Generator().manual_seed(1)).int().view(2, 6).cuda()
    kc = torch.zeros((12, page, G, D), dtype=dtype, device="cuda")
    vc = torch.zeros_like(kc)
    ang = torch.rand((room, D // 2), device="cuda") * 6.3
    cos, sin = ang.cos(), ang.sin()
    past = [0, 0]
    dense = [None, None]
    for new in ([19, 33], [1, 1], [1, 1], [2, 1], [1, 3], [1, 1], [1, 1]):
        n = sum(new)
        qkv = torch.randn((n, (heads + 2 * G) * D), device="cuda")
        q, k, v = qkv.split([heads * D, G * D, G * D], 1)
        cu = torch.tensor([0, new[0], n], dtype=torch.int32, device="cuda")
        pt = torch.tensor(past, dtype=torch.int32, device="cuda")
        values = dict(q=qkv if packed else q, k=k, v=v, kc=kc, vc=vc, cu=cu, past=pt, bt=table,
                      cos=cos, sin=sin)
        ins = ["q", "", ""] if packed else ["q", "k", "v"]
        out, key_out, value_out = sess.dispatch(
            dict(op_type="PagedAttention",
                 inputs=ins + ["kc", "vc", "cu", "past", "bt", "cos", "sin"],
                 attrs=dict(num_heads=heads, kv_num_heads=G, do_rotary=1)), values)
        assert key_out is kc and value_out is vc
        start = 0
        for b in range(2):
            rows = slice(start, start + new[b])
            if dtype == F32:
                pk, pv = dense[b] or (None, None)
                want, pk, pv = sess.group_query_attention(
                    q[None, rows], k[None, rows], v[None, rows], heads, G, do_rotary=True,
                    cos_cache=cos, sin_cache=sin, past_key=pk, past_value=pv)
                dense[b] = (pk, pv)
                near(want[0], out[rows], 2 * TOL)  # each side may be off by TOL
            start += new[b]
        pos = torch.cat([torch.arange(p, p + m) for p, m in zip(past, new)]).cuda()
        rot = ref.rotate(q.reshape(n, heads, D), cos[pos], sin[pos], False).float().view(n, -1)
        s = dict(key=kc, value=vc, table=table, cu=cu, past=pt, q=rot)
        near(ref.attention(s, new, past, heads), out)
        past = [p + m for p, m in zip(past, new)]
    sess.sync()
