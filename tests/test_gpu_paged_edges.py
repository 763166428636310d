"""The paged KV cache at its edges: many heads a group, extreme values, lengths
that fall, destroyed streams.  Formulas and tolerances as in
tests/test_gpu_paged.py.
"""
import math

import pytest
import torch

from tests import paged_reference as ref
from tests.test_gpu_paged import BF16, F16, F32, handle, near, reported, run, sess  # noqa: F401,E501

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads", [71, 128, 130])
@pytest.mark.parametrize("new,past,window,shared", [
    ([1], [200], 0, 0), ([40, 1, 3], [5, 300, 0], 0, 0), ([7, 1], [300, 400], 0, 257),
    ([90], [30], 50, 0)])
def test_more_heads_than_a_tile_has_rows(sess, heads, new, past, window, shared, dtype):
    """All query heads on one KV head: a token's heads lie in several tiles of 16 rows."""
    s = ref.make(30, dtype, new, past, heads, 1, 64, 16, shared)
    want = ref.attention(s, new, past, heads, window=window)
    near(want, run(sess, s, heads, new, local_window_size=window, shared_len=shared))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("scale", [1, 60])  # few rows, and tiles of 128
@pytest.mark.parametrize("cu,kept", [
    ([0, 10, 2, 5, 8], 0),    # a sequence behind the fall would share tokens 5 to 7
    ([0, 3, 2, 5, 9], 1),
    ([0, 3, 5, 4, 9], 2),
    ([0, 3, 5, 9, 8], 2),     # the third passes the last length
    ([0] * 300 + [3, 2, 5, 9], 300)])
def test_lengths_that_fall_leave_out_what_lies_behind(sess, cu, kept, scale, dtype):
    """Sequences before the fall keep their results; no row of another is written, and
    nothing of them is appended."""
    heads, G, D, past = 8, 2, 64, 50
    batch = len(cu) - 1
    cu = [scale * x for x in cu]
    new = [b - a if i < kept else 0 for i, (a, b) in enumerate(zip(cu, cu[1:]))]
    s = ref.make(31, dtype, new, [past] * batch, heads, G, D, 16, garbage=False)
    n = 9 * scale
    q = torch.randn((n, heads * D), device="cuda")
    s = {**s, "q": q, "cu": torch.tensor(cu, dtype=torch.int32, device="cuda"),
         "table": s["table"].clamp_min(0)}
    good = sum(new)
    want = ref.attention({**s, "q": q[:good]}, new, [past] * batch, heads)
    for shared in (0, 16):
        if shared:  # one prefix for all: sequence 0's first page
            s["table"][:, 0] = s["table"][0, 0]
            want = ref.attention({**s, "q": q[:good]}, new, [past] * batch, heads)
        out = torch.full_like(q, 7.0)
        run(sess, s, heads, new, checked=False, out=out, max_seq=n, shared_len=shared)
        if good:
            near(want, out[:good])
        assert (out[good:] == 7.0).all()
        reported(sess, "cu_seqlens")
    kv = torch.randn((n, G * D), device="cuda")
    key, value = s["key"].clone(), s["value"].clone()
    out = torch.full_like(q, 7.0)
    sess.paged_kv_append(handle(s), kv, kv, q=q, num_heads=heads, q_out=out)
    reported(sess, "cu_seqlens")
    assert torch.equal(out[:good], q[:good]) and (out[good:] == 7.0).all()
    row = 0
    for b, m in enumerate(new):
        pos = torch.arange(past, past + m)
        where = (s["table"][b].cpu()[pos // 16].long(), pos % 16)
        for cache in (key, value):
            cache[where] = kv[row:row + m].view(m, G, D).to(dtype)
        row += m
    assert torch.equal(key, s["key"]) and torch.equal(value, s["value"])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size", [2.0 ** 23, 1e8, 1e12])
@pytest.mark.parametrize("new,past,shared", [([1, 3], [90, 200], 0), ([140, 60], [0, 33], 0),
                                             ([1, 150], [90, 200], 80)])
def test_scores_that_leave_one_key(sess, new, past, shared, size, dtype):
    """Scores so large that a row's weight is all on its largest.  Scores are held to
    2^-20 of sum |q k| at least; rows whose two largest lie 2^-16 of it apart (near all)
    give that key's value."""
    heads, G, D = 8, 2, 64
    s = ref.make(32, dtype, new, past, heads, G, D, 16, shared)
    s["q"] *= size
    want = ref.attention(s, new, past, heads)
    got = run(sess, s, heads, new, shared_len=shared)
    assert torch.isfinite(got).all()
    clear = torch.zeros((sum(new), heads), dtype=torch.bool)
    row = 0
    for b, (n, p0) in enumerate(zip(new, past)):
        pos = torch.arange(n + p0)
        k = s["key"][s["table"][b].cpu()[pos // 16].long(), pos % 16].double()
        for i in range(n):
            q = s["q"][row].double().view(G, heads // G, D)
            sc = torch.einsum("ghd,tgd->ght", q, k[:p0 + i + 1])
            size_of = torch.einsum("ghd,tgd->ght", q.abs(), k[:p0 + i + 1].abs()).amax(-1)
            if p0 + i:
                top = sc.topk(2, -1).values
                clear[row] = (top[..., 0] - top[..., 1] > 2.0 ** -16 * size_of).flatten().cpu()
            else:
                clear[row] = True
            row += 1
    assert clear.float().mean() > 0.99
    clear = clear.cuda()
    near(want.view(-1, heads, D)[clear], got.view(-1, heads, D)[clear])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("page", [16, 12])  # TMA boxes, copies of 16 bytes
@pytest.mark.parametrize("new,past,window", [([140, 90], [900, 700], 0), ([1, 2], [900, 700], 0),
                                             ([150, 40], [900, 700], 300)])
def test_missing_pages_inside_what_all_rows_see(sess, new, past, window, page, dtype):
    """Keys of a page that is not there are left out of blocks that every row sees, and the
    rows' own keys behind them are not."""
    heads, G, D = 8, 2, 64
    s = ref.make(33, dtype, new, past, heads, G, D, page)
    want = torch.zeros((sum(new), heads, D), dtype=torch.float64, device="cuda")
    bad = {b: [p // page - 30 + b, p // page - 7, p // page - 12] for b, p in enumerate(past)}
    row = 0
    for b, (n, p0) in enumerate(zip(new, past)):
        pos = torch.arange(n + p0, device="cuda")
        where = (s["table"][b][pos // page].long(), pos % page)
        k, v = s["key"][where].double(), s["value"][where].double()
        gone = torch.isin(pos // page, torch.tensor(bad[b], device="cuda"))
        for i in range(n):
            q = s["q"][row].double().view(G, heads // G, D)
            sc = torch.einsum("ghd,tgd->ght", q, k) / math.sqrt(D)
            hide = gone | (pos > p0 + i)
            if window:
                hide = hide | (pos <= p0 + i - window)
            weight = torch.softmax(sc.masked_fill(hide, -math.inf), -1)
            want[row] = torch.einsum("ght,tgd->ghd", weight, v).reshape(heads, D)
            row += 1
    for b, pages in bad.items():
        for p, x in zip(pages, (-3, 2 ** 30, s["key"].shape[0])):
            s["table"][b, p] = x
    got = run(sess, s, heads, new, checked=False, local_window_size=window)
    near(want.flatten(1), got)
    reported(sess, "page")


def test_workspace_grows_while_another_stream_is_captured(sess):
    """A call outside the capture, on a stream whose workspace is too small for it, in a
    thread that captures another stream (in the mode that forbids the most)."""
    small = ref.make(34, F16, [1], [300], 8, 2, 64, 16)
    large = ref.make(35, F16, [200, 90], [100, 700], 8, 2, 64, 16)
    want_small, want_large = run(sess, small, 8, [1]), run(sess, large, 8, [200, 90])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(sess, small, 8, [1])
    out, h = torch.zeros_like(large["q"]), handle(large)
    got, hs = torch.zeros_like(small["q"]), handle(small)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="global"):
        sess.paged_attention(hs, small["q"], 8, max_seq=1, out=got)
        with torch.cuda.stream(side):
            sess.paged_attention(h, large["q"], 8, max_seq=200, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want_large) and torch.equal(got, want_small)
    sess.sync()


def test_stream_destroyed_with_work_to_run_and_its_handle_used_again(sess):
    """Work of a destroyed stream still runs; the next stream may get its handle, and must
    not get its workspace while that is so."""
    import ctypes
    rt = ctypes.CDLL("libcudart.so.12")

    def create():
        p = ctypes.c_void_p()
        assert rt.cudaStreamCreateWithFlags(ctypes.byref(p), 1) == 0
        return p.value

    cases = []
    for i, (new, past) in enumerate((([1] * 3, [9000] * 3), ([1] * 8, [4000] * 8))):
        s = ref.make(36 + i, F16, new, past, 8, 2, 128, 16)
        cases.append((s, handle(s), run(sess, s, 8, new), torch.zeros_like(s["q"])))
    (s0, h0, want0, out0), (s1, h1, want1, out1) = cases
    outs = [torch.zeros_like(out1) for _ in range(30)]
    torch.cuda.synchronize()
    first, others = create(), []
    try:
        sess.set_stream(first)
        with torch.cuda.stream(torch.cuda.ExternalStream(first)):
            torch.cuda._sleep(40_000_000)  # some 20 ms
        sess.paged_attention(h0, s0["q"], 8, max_seq=1, out=out0)
        assert rt.cudaStreamDestroy(ctypes.c_void_p(first)) == 0
        while first not in others and len(others) < 16:
            others.append(create())
        sess.set_stream(others[-1])
        for out in outs:
            sess.paged_attention(h1, s1["q"], 8, max_seq=1, out=out)
        torch.cuda.synchronize()
        sess.sync()
        assert torch.equal(out0, want0)
        assert all(torch.equal(out, want1) for out in outs)
    finally:
        sess.set_stream(None)
        for p in others:
            rt.cudaStreamDestroy(ctypes.c_void_p(p))


@pytest.mark.parametrize("new", [[1, 2], [80, 70]])
def test_lengths_and_pages_are_reported_together(sess, new):
    s = ref.make(38, F16, new, [300, 400], 8, 2, 64, 16)
    s["table"][0, 3] = -1
    s["past"][1] = -1
    run(sess, s, 8, new, checked=False)
    with pytest.raises(ValueError, match="cu_seqlens.*block_table"):
        sess.sync()
    sess.sync()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,past", [([1, 3], [90, 200]), ([140, 60], [0, 33])])
@pytest.mark.parametrize("scale,softcap,size", [
    (None, 2.0 ** 20, 1.0), (None, 2.0 ** 20, 2.0 ** 24), (0.125, 2.0 ** -20, 1.0),
    (2.0 ** -100, 0.0, 2.0 ** 97), (2.0 ** -100, 30.0, 2.0 ** 97)])
def test_extreme_scales_and_caps(sess, scale, softcap, size, new, past, dtype):
    """At the ends of what is taken.  A cap of 2^-20 leaves the mean; scores behind a cap of
    2^20 are held to its last bits in fp32 (2^-4), so the sharp rows there have to be finite
    and of a value's size only."""
    s = ref.make(39, dtype, new, past, 8, 2, 64, 16)
    s["q"] *= size
    got = run(sess, s, 8, new, scale=scale, softcap=softcap)
    want = ref.attention(s, new, past, 8, scale, softcap)
    if softcap == 2.0 ** 20 and size > 1:
        assert torch.isfinite(got).all()
        assert got.abs().max() <= s["value"].float().nan_to_num().abs().max() * (1 + 1e-5)
    else:
        near(want, got)


def test_scales_and_caps_that_fp32_does_not_hold_are_refused(sess):
    s = ref.make(15, F16, [2], [5], 8, 2, 64, 16)
    for kw in (dict(scale=1e300), dict(scale=1e-300), dict(softcap=1e300), dict(softcap=1e-300),
               dict(softcap=1e7), dict(softcap=1e-7), dict(scale=1e-38), dict(scale=1e38)):
        with pytest.raises(ValueError, match="lies in"):
            sess.paged_attention(handle(s), s["q"], 8, **kw)


def test_append_of_a_token_that_32_bits_do_not_count_is_refused(sess):
    """The features of a token's q, k and v rows together pass 2^31 (checked without tokens:
    nothing is launched)."""
    import ctypes
    from onnx_runtime_dart_b200 import _lib
    G, D, some = 1 << 24, 64, torch.zeros(4, device="cuda").data_ptr()
    c = _lib.PagedCacheStruct(some, some, some, some, some, 1, 1, 1, 1, D, G, _lib.CACHE_F16)
    for heads, rc in ((0, _lib.ERR_INVALID_ARG), (G, _lib.ERR_INVALID_ARG), (None, 0)):
        kv = 1 << 23 if heads is None else G
        c.kv_num_heads = kv
        q = some if heads else 0
        assert _lib.load().ort_cuda_paged_kv_append(
            sess.handle, ctypes.addressof(c), q, (heads or 0) * D, some, kv * D, some, kv * D, 0,
            heads or 0, 0, 0, 0, 0, q, 0) == rc


@pytest.mark.parametrize("dtype", [F32, F16])
def test_outputs_in_the_pages_are_refused(sess, dtype):
    s = ref.make(40, dtype, [2], [5], 8, 2, 64, 16, garbage=False)
    h, kv = handle(s), torch.zeros((2, 128), device="cuda")
    for pages in (s["key"], s["value"]):
        out = pages.view(torch.uint8).flatten()[-4096:].view(torch.float32).view(2, 512)
        with pytest.raises(ValueError, match="overlaps the pages"):
            sess.paged_attention(h, s["q"], 8, out=out)
        with pytest.raises(ValueError, match="overlaps the pages"):
            sess.paged_kv_append(h, kv, kv, q=s["q"], num_heads=8, q_out=out)
    same = {**s, "value": s["key"]}
    with pytest.raises(ValueError, match="same pages"):
        sess.paged_kv_append(handle(same), kv, kv)
    near(ref.attention(same, [2], [5], 8), run(sess, same, 8, [2]))  # reading them is fine


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,past", [([1, 3], [600, 300]), ([140, 90], [600, 300])])
@pytest.mark.parametrize("plant", [math.inf, -math.inf, math.nan])
def test_values_a_row_sees_that_are_not_finite(sess, new, past, plant, dtype):
    """They make the feature they stand in not finite in the rows that see them, deep inside
    the sequence and at the border of the mask, and touch no other feature."""
    heads, G, D = 8, 2, 64
    s = ref.make(41, dtype, new, past, heads, G, D, 16)
    want = ref.attention(s, new, past, heads).view(-1, heads, D)
    seen = torch.zeros_like(want, dtype=torch.bool)
    row = 0
    for b, (n, p0) in enumerate(zip(new, past)):
        for j, d in ((130 + b, 3), (p0, 17), (p0 + n - 1, 40)):
            s["value"][int(s["table"][b, j // 16]), j % 16, :, d] = plant
            seen[row + max(0, j - p0):row + n, :, d] = True
        row += n
    got = run(sess, s, heads, new).view(-1, heads, D)
    assert not torch.isfinite(got[seen]).any()
    near(want[~seen], got[~seen])


def test_query_rows_that_are_not_finite(sess):
    """They stay in their row."""
    for dtype in (F32, F16, BF16):
        for new, past in (([1, 3], [600, 300]), ([140, 90], [600, 300])):
            s = ref.make(42, dtype, new, past, 8, 2, 64, 16)
            want = ref.attention(s, new, past, 8)
            s["q"][0], s["q"][2, 100] = math.nan, math.inf
            got = run(sess, s, 8, new)
            keep = torch.ones_like(got, dtype=torch.bool)
            keep[0] = keep[2, 64:128] = False
            near(want[keep], got[keep])
            assert got[0].isnan().all() and not torch.isfinite(got[2, 64:128]).any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lead", [0, 1])  # 16-byte pieces, and the kernel for any alignment
def test_append_rounds_once(sess, dtype, interleaved, lead):
    """Keys whose rotation lies next to the middle of two 16-bit numbers, where fp32 holds
    the middle only: the nearest of the two all the same.  And keys drawn at random."""
    import numpy as np
    n, G, D, half = 64, 2, 128, 64
    bits = 11 if dtype == F16 else 8
    g = torch.Generator().manual_seed(43)
    r = torch.randint(2 ** (bits - 1), 2 ** bits, (n // 2, G * D), generator=g).double() + 0.5
    middle = r * 2.0 ** -(bits - 1) * (torch.randint(0, 2, r.shape, generator=g) * 2 - 1)
    k = torch.cat([middle, torch.randn((n // 2, G * D), generator=g).double()]).float()
    assert torch.equal(k[:n // 2].double(), middle)
    ang = torch.rand((n, half), generator=g, dtype=torch.float64) * 6.3
    cos, sin = ang.cos().float(), ang.sin().float()
    cos[:n // 2], sin[:n // 2] = 1.0, 2.0 ** -30
    s = ref.make(44, dtype, [n], [0], 2, G, D, 16)
    fused = torch.zeros((n, G * D + 4 * lead), device="cuda")
    rows = fused[:, lead:lead + G * D] if lead else fused
    rows.copy_(k)
    sess.paged_kv_append(handle(s), rows, rows, cos_cache=cos.cuda(), sin_cache=sin.cuda(),
                         rotary_interleaved=interleaved)
    sess.sync()
    want = ref.rotate(k.view(n, G, D), cos, sin, interleaved)  # exact in the rows of middles
    pos = torch.arange(n)
    have = s["key"][s["table"][0].cpu()[pos // 16].long(), pos % 16].cpu()
    word = have.view(torch.int16)
    off = (have.double() - want).abs()
    for step in (-1, 1):  # the neighbours
        other = (word + step).view(dtype).double()
        away = (other - want).abs()
        assert (off[:n // 2] < away[:n // 2]).all()
        assert (off[n // 2:] <= away[n // 2:] * (1 + 1e-9)).all()
    assert np.isfinite(have.double().numpy()).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,past", [([1, 1, 1], [200, 40, 9]), ([90, 1, 33], [20, 300, 0])])
@pytest.mark.parametrize("attrs", [dict(local_window_size=1), dict(local_window_size=37),
                                   dict(softcap=3.0), dict(scale=0.5),
                                   dict(scale=0.05, softcap=20.0, local_window_size=64)])
def test_dispatch_hands_on_the_attributes(sess, new, past, attrs, dtype):
    """A window of w keys has the query's own among them: w = 1 gives the key's own value."""
    heads, G, D, n = 8, 2, 64, sum(new)
    s = ref.make(45, dtype, new, past, heads, G, D, 16)
    k, v = (torch.randn((n, G * D), device="cuda") for _ in range(2))
    out, key, value = sess.dispatch(
        dict(op_type="PagedAttention", inputs=["q", "k", "v", "kc", "vc", "cu", "past", "bt"],
             attrs=dict(num_heads=heads, kv_num_heads=G, **attrs)),
        dict(q=s["q"], k=k, v=v, kc=s["key"], vc=s["value"], cu=s["cu"], past=s["past"],
             bt=s["table"]))
    sess.sync()
    want = ref.attention(s, new, past, heads, attrs.get("scale"), attrs.get("softcap", 0.0),
                         attrs.get("local_window_size", 0))
    near(want, out)
    if attrs == dict(local_window_size=1):
        own = v.to(dtype).double().view(n, G, 1, D).expand(n, G, heads // G, D).reshape(n, -1)
        near(own, out)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("head", [8, 24, 48, 104])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (4, 1)])
def test_small_and_odd_heads_on_whole_pages(sess, head, heads, kv_heads, dtype):
    """Heads narrower than a box of a page, prompts and single tokens."""
    new, past = [150, 1], [20, 300]
    s = ref.make(46, dtype, new, past, heads, kv_heads, head, 16)
    near(ref.attention(s, new, past, heads), run(sess, s, heads, new))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("window", [2 ** 31 - 2, 2 ** 31 - 1, 2 ** 40])
def test_windows_longer_than_any_sequence(sess, window, dtype):
    for new, past, shared in (([150, 1], [20, 300], 0), ([150, 1], [20, 300], 17), ([1], [9], 0)):
        s = ref.make(47, dtype, new, past, 8, 2, 64, 16, shared)
        near(ref.attention(s, new, past, 8),
             run(sess, s, 8, new, local_window_size=window, shared_len=shared))


@pytest.mark.parametrize("dtype", [F32, F16])
def test_output_at_an_odd_address(sess, dtype):
    for new, past, shared in (([150, 1], [20, 300], 0), ([90, 2], [20, 300], 17), ([1], [9], 0)):
        s = ref.make(48, dtype, new, past, 8, 2, 64, 16, shared)
        n = s["q"].numel()
        out = torch.full((n + 2,), 7.0, device="cuda")
        run(sess, s, 8, new, shared_len=shared, out=out[1:-1].view(-1, 512))
        near(ref.attention(s, new, past, 8), out[1:-1].view(-1, 512))
        assert out[0] == 7.0 and out[-1] == 7.0


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("shared", [0, 16])
def test_call_whose_sequences_are_all_empty(sess, shared, dtype):
    """A padded step without a token in it: nothing is written, nothing reported."""
    s = ref.make(49, dtype, [0, 0, 0], [40, 20, 16], 8, 2, 64, 16, shared)
    for n in (1, 200):
        q = torch.full((n, 512), math.nan, device="cuda")
        out = torch.full_like(q, 7.0)
        run(sess, {**s, "q": q}, 8, [n], out=out, shared_len=shared)
        assert (out == 7.0).all()


def test_captured_step_follows_a_batch_that_falls_apart_and_recovers(sess):
    """Replays of one captured call over lengths that fit, fall, and fit again."""
    new, past, heads = [70, 1, 40], [100, 300, 5], 8
    s = ref.make(50, F16, new, past, heads, 2, 64, 16)
    want = run(sess, s, heads, new)
    good = s["cu"].clone()
    out, h = torch.zeros_like(s["q"]), handle(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sess.paged_attention(h, s["q"], heads, max_seq=70, out=out)
    for _ in range(3):
        out.fill_(7.0)
        s["cu"].copy_(good)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        sess.sync()
        out.fill_(7.0)
        s["cu"][2] = 3
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:70], want[:70]) and (out[70:] == 7.0).all()
        reported(sess, "cu_seqlens")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,past,shared,window", [
    ([1, 2], [40, 90], 0, 0), ([130, 70], [40, 90], 0, 30), ([130, 3], [40, 90], 33, 0),
    ([1, 2], [40, 90], 33, 60)])
def test_tokens_before_the_first_sequence_are_padding(sess, new, past, shared, window, dtype):
    heads, G, D, lead = 8, 2, 64, 9
    s = ref.make(51, dtype, new, past, heads, G, D, 16, shared)
    want = ref.attention(s, new, past, heads, window=window)
    q = torch.cat([torch.full((lead, heads * D), math.nan, device="cuda"), s["q"]])
    t = {**s, "q": q, "cu": s["cu"] + lead}
    out = torch.full_like(q, 7.0)
    run(sess, t, heads, new, out=out, shared_len=shared, local_window_size=window)
    near(want, out[lead:])
    assert (out[:lead] == 7.0).all()
    kv = torch.randn((len(q), G * D), device="cuda")
    kv[:lead] = math.nan
    before = s["key"].isnan().sum()
    sess.paged_kv_append(handle(t), kv, kv)
    sess.sync()
    assert s["key"].isnan().sum() == before
    page = int(s["table"][0, past[0] // 16])
    assert torch.equal(s["key"][page, past[0] % 16].flatten(), kv[lead].to(dtype))
