"""The token-step operators at the values and uses where they can go wrong: infinities beside masked places, exact products, eps 0, tensors that
carry gradients, several callers of one handle.  Plain implementations and bounds as in test_gpu_ops.py."""
import math

import pytest
import torch

from test_gpu_ops import ACT, U32, Layer, Paged, ints, ops, rnd, u  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------------------------
# attention
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv,rep", [(1, 1), (2, 2), (1, 4), (2, 7)])
@pytest.mark.parametrize("lens,window", [([21, 32, 1, 129], 0), ([33, 70, 500, 31], 27), ([3000, 45, 1, 1027], 0), ([3000, 2011], 1999)])
def test_attention_of_an_infinity_in_a_32_bit_cache(ops, hd, kv, rep, lens, window):  # noqa: F811
    """A 32-bit cache keeps its values: an infinity that is seen is the result of its column, and no other column, head or sequence changes.  It
    stands in the last token, the first that is seen, and one between; the places behind and before are masked."""
    P = Paged(ops, lens, kv, hd, 16, "f32", seed=hd + rep)
    q = rnd((len(lens), kv * rep, hd), torch.float32, 5).cuda()
    want, lse = ops.attention(q, P.cache, P.table, P.lens_dev, window=window, lse=True)
    ops.sync()
    assert bool(want.isfinite().all())
    for b, n in enumerate(lens):
        low = max(0, n - window) if window else 0
        for i, t in enumerate({n - 1, low, (low + n) // 2}):
            page, head, col = int(P.table[b, t // 16]), (i + 1) % kv, (7 * i + 3) % hd
            kept = float(P.cache.v[page, head, t % 16, col])
            P.cache.v[page, head, t % 16, col] = -math.inf if i == 1 else math.inf
            out, got = ops.attention(q, P.cache, P.table, P.lens_dev, window=window, lse=True)
            ops.sync()
            P.cache.v[page, head, t % 16, col] = kept
            expect = want.clone()
            expect[b, head * rep:(head + 1) * rep, col] = -math.inf if i == 1 else math.inf
            assert torch.equal(out, expect) and torch.equal(got, lse), (b, t)


@pytest.mark.parametrize("act,store,lens", [("bf16", "same", [300, 0, 33]), ("bf16", "same", [5000, 0, 2100]), ("f16", "int8", [3000, 1, 900]), ("f32", "same", [300, 0, 33]),
                                            ("f32", "same", [5000, 0, 2100]), ("f32", "e4m3", [40, 2, 900])])
def test_attention_in_place(ops, act, store, lens):  # noqa: F811
    """out may be q: a query head's row is read by the workgroups that write it, or written by the join behind all that read it."""
    P = Paged(ops, lens, 2, 64, 16, act, store, seed=3)
    q = rnd((3, 34, 64), ACT[act], 4).cuda()
    want = ops.attention(q, P.cache, P.table, P.lens_dev)
    for _ in range(5):
        into = q.clone()
        assert ops.attention(into, P.cache, P.table, P.lens_dev, out=into).data_ptr() == into.data_ptr()
        assert torch.equal(into, want)
    ops.sync()


def test_a_sync_inside_a_capture_is_refused(pkg, ops):  # noqa: F811
    """... and the capture goes on."""
    x, w = torch.zeros((2, 64), device="cuda"), torch.ones(64, device="cuda")
    ops.add_rmsnorm(x, w)
    ops.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = ops.add_rmsnorm(x, w)[1]
        with pytest.raises(pkg.HipVocError) as e:
            ops.sync()
        b = ops.add_rmsnorm(a, w)[1]
    assert e.value.code == -1 and "captured" in str(e.value)
    for rep in range(3):
        x.copy_(rnd((2, 64), torch.float32, rep))
        one = ops.add_rmsnorm(x, w)[1]
        two = ops.add_rmsnorm(one, w)[1]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, one) and torch.equal(b, two)
    ops.sync()


# ---------------------------------------------------------------------------------------------------------------------
# several callers
def test_syncs_do_not_wait_for_each_other(pkg, ops):  # noqa: F811
    """While one thread waits for a stream that is busy, others that wait for idle ones return.  A stream may stand behind the busy one in the same hardware
    queue, and the runtime has locks of its own, so it is enough that one of six returns early in one of five rounds; behind a lock none ever does."""
    import threading
    import time
    busy, idle = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(6)]
    handles = [pkg.HipOps.open(0) for _ in range(3)] + [ops] * 3
    torch.cuda._sleep(1000)
    ended = {}

    def wait(name, s, h):
        with torch.cuda.stream(s):
            h.sync()
        ended[name] = time.perf_counter()
    for i, (s, h) in enumerate(zip([busy] + idle, [ops] + handles)):       # everything is loaded and warm
        wait(i, s, h)
    for _ in range(5):
        with torch.cuda.stream(busy):
            torch.cuda._sleep(2_000_000_000)                    # about 0.8 s, then it ends
        threads = [threading.Thread(target=wait, args=(i, s, h)) for i, (s, h) in enumerate(zip([busy] + idle, [ops] + handles))]
        threads[0].start()
        time.sleep(0.1)                                         # the first one is waiting by now
        for t in threads[1:]:
            t.start()
        for t in threads:
            t.join()
        if any(ended[i] < ended[0] - 0.2 for i in range(1, 7)):
            break
    else:
        pytest.fail(f"all waited: {ended}")
    for h in handles[:3]:
        h.close()


def test_whose_errors_a_sync_reports(pkg, ops):  # noqa: F811
    """One handle: the first sync behind the call reports it, whichever stream it waits for, and no other.  A handle each: the one whose call it was."""
    P = Paged(ops, [40, 9], 1, 64, 8, "bf16", seed=3)
    q = rnd((2, 2, 64), torch.bfloat16, 4).cuda()
    bad = P.table.clone()
    bad[0, 2] = P.cache.n_pages
    torch.cuda.synchronize()
    for one in (True, False):
        mine, other = (ops, ops) if one else (ops, pkg.HipOps.open(0))
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        with torch.cuda.stream(streams[0]):
            good = mine.attention(q, P.cache, P.table, P.lens_dev)
        with torch.cuda.stream(streams[1]):
            wrong = other.attention(q, P.cache, bad, P.lens_dev)
        torch.cuda.synchronize()
        raised = []
        for s, h in zip(streams, (mine, other)):
            with torch.cuda.stream(s):
                try:
                    h.sync()
                    raised.append(False)
                except pkg.HipVocError as e:
                    raised.append(e.code == -2 and "page" in str(e))
        assert raised == [one, not one]
        assert bool(good.isfinite().all()) and bool(wrong[0].isnan().all()) and torch.equal(wrong[1], good[1])
        ops.sync()
        other.sync()
        if not one:
            other.close()


def test_many_syncs_at_once(pkg, ops):  # noqa: F811
    """More waiting threads than the handle has words: each gets one in its turn, and one error is reported once."""
    import threading
    P = Paged(ops, [40], 1, 64, 8, "bf16", seed=5)
    q = rnd((1, 2, 64), torch.bfloat16, 4).cuda()
    bad = P.table.clone()
    bad[0, 2] = -3
    ops.attention(q, P.cache, bad, P.lens_dev)
    torch.cuda.synchronize()
    seen, lock = [], threading.Lock()

    def run():
        for _ in range(20):
            try:
                ops.sync()
                code = 0
            except pkg.HipVocError as e:
                code = e.code
            with lock:
                seen.append(code)
    threads = [threading.Thread(target=run) for _ in range(100)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(seen) == 2000 and sorted(seen)[:2] == [-2, 0]


def test_texts_of_refusals_from_several_threads(pkg, ops):  # noqa: F811
    """What the vocoder's and the encoder's entry points say to an operator handle is written like its own refusals: every text read is a whole one."""
    import threading
    L = ops._L
    enc = pkg.encoder._lib()
    other = "this handle is an operator handle (hipvoc_ops_open)"
    assert L.hipvoc_decode(ops._h, None, 0, None, 0, None) == -1 and L.hipvoc_last_error(ops._h).decode() == other
    assert L.hipvoc_ops_sync(ops._h, None) == 0
    assert enc.hipvoc_enc_encode_batch(ops._h, None, None, 0, None, None, None) == -1 and L.hipvoc_last_error(ops._h).decode() == other
    x, w = torch.zeros((2, 64), device="cuda"), torch.ones(64, device="cuda")
    texts = {other, "eps must be finite and not negative", "group 7 must be 0, or for 8-bit rows 32, 64 or 128 and a divisor of cols 64"}
    wrong = []

    def run(i):
        for _ in range(400):
            if i % 3 == 0:
                L.hipvoc_decode(ops._h, None, 0, None, 0, None)
            elif i % 3 == 1:
                enc.hipvoc_enc_encode_batch(ops._h, None, None, 0, None, None, None)
            else:
                try:
                    ops.add_rmsnorm(x, w, **({"eps": -1.0} if i == 2 else {"group": 7}))
                    wrong.append("not refused")
                except pkg.HipVocError as e:
                    if not any(t in str(e) for t in texts):
                        wrong.append(str(e))
            if L.hipvoc_last_error(ops._h).decode() not in texts:
                wrong.append("text")
    threads = [threading.Thread(target=run, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


# ---------------------------------------------------------------------------------------------------------------------
# tensors that are more than their memory
def test_gradients_are_refused_not_dropped(pkg, ops):  # noqa: F811
    """There is no backward: a tensor that requires a gradient is refused while gradients are recorded, and taken under no_grad or inference_mode."""
    P = Paged(ops, [9, 12], 2, 64, 8, "bf16", seed=1)
    new, cu, first = rnd((2, 2, 64), torch.bfloat16, 1).cuda(), ints([0, 1, 2]), ints([8, 11])
    q, x, w = rnd((2, 4, 64), torch.bfloat16, 1).cuda(), rnd((2, 64), torch.bfloat16, 2).cuda(), rnd((64,), torch.bfloat16, 3).cuda()
    codes, scales = torch.randint(0, 256, (8, 32), dtype=torch.uint8, device="cuda"), torch.ones((8, 2), dtype=torch.float16, device="cuda")
    grad = lambda t: t.detach().clone().requires_grad_()  # noqa: E731
    calls = {
        "q": (lambda t: ops.attention(t, P.cache, P.table, P.lens_dev), q),
        "out": (lambda t: ops.attention(q, P.cache, P.table, P.lens_dev, out=t), q),
        "k": (lambda t: ops.kv_write(P.cache, t, new, P.table, cu, first), new),
        "v": (lambda t: ops.kv_write(P.cache, new, t, P.table, cu, first), new),
        "x": (lambda t: ops.add_rmsnorm(t, w, x), x),
        "weight": (lambda t: ops.add_rmsnorm(x, t), w),
        "residual": (lambda t: ops.add_rmsnorm(x, w, t), x),
        "x ": (lambda t: ops.q4_matvec(codes, scales, t), x),
        "scales": (lambda t: ops.q4_matvec(codes, t, x), scales),
        "mins": (lambda t: ops.q4_matvec(codes, scales, x, mins=t), scales),
    }
    for name, (call, t) in calls.items():
        leaf = grad(t)
        for kind in (leaf, leaf * 1):
            with pytest.raises(pkg.HipVocError) as e:
                call(kind)
            assert e.value.code == -1 and str(e.value).strip().split("requires grad")[0].endswith(name.strip() + " "), str(e.value)
            with torch.no_grad():
                call(kind)
            with torch.inference_mode():
                call(kind)
            call(kind.detach())
    ops.sync()


def test_views_of_a_negative_are_refused(pkg, ops):  # noqa: F811
    """The imaginary part of a conjugate is a real tensor whose memory holds its negative."""
    z = torch.view_as_complex(rnd((2, 64, 2), torch.float32, 1).cuda()).conj().imag
    assert z.is_neg() and z.dtype == torch.float32
    flat = torch.empty_strided((2, 64), (64, 1), device="cuda")
    neg = torch._neg_view(flat)
    with pytest.raises(pkg.HipVocError) as e:
        ops.add_rmsnorm(neg, torch.ones(64, device="cuda"))
    assert e.value.code == -1 and "negative" in str(e.value)
    ops.add_rmsnorm(neg.resolve_neg(), torch.ones(64, device="cuda"))
    ops.sync()


# ---------------------------------------------------------------------------------------------------------------------
# norm
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", [5, 96, 640, 2056, 40000])
def test_add_rmsnorm_with_eps_0(ops, act, cols):  # noqa: F811
    """A row of zeros has no norm without eps: NaN, in 8 bits by its scale.  Its neighbours keep theirs."""
    x = rnd((3, cols), ACT[act], cols).cuda()
    w = (1 + 0.1 * rnd((cols,), torch.float32, 1)).to(ACT[act]).cuda()
    x[1] = 0
    zero = torch.zeros_like(x)
    for res in (None, zero):
        total, y = ops.add_rmsnorm(x, w, res, eps=0.0)
        alone = ops.add_rmsnorm(x[::2].contiguous(), w, None, eps=0.0)[1]
        assert bool(y[1].isnan().all()) and torch.equal(y[::2], alone) and bool(alone.isfinite().all())
        assert res is None or torch.equal(total, x)
        for quant in ("int8", "e4m3"):
            for group in (0, 32):
                if cols % (group or 1):
                    continue
                _, codes, scales = ops.add_rmsnorm(x, w, res, eps=0.0, quant=quant, group=group)
                assert bool(scales[1].isnan().all()) and bool(scales[::2].isfinite().all()) and bool((codes[1].float() == 0).all())
                back = codes.float().reshape(3, -1, group or cols) * scales[..., None]
                assert bool(back[1].isnan().all()) and bool(back[::2].isfinite().all())
    ops.sync()


# ---------------------------------------------------------------------------------------------------------------------
# 4-bit products
Q4_SHAPES = [  # weight rows, group, groups, x rows: each kernel and tile count, whole slabs of 128 columns and not, at and over 128 groups
    (17, 32, 1, 1), (33, 64, 3, 2), (100, 32, 129, 5), (70, 32, 257, 17), (300, 128, 130, 3), (4100, 64, 9, 3), (8190, 32, 131, 1), (8193, 32, 260, 2), (2050, 64, 17, 40),
    (16390, 32, 33, 17), (16385, 32, 131, 5), (65541, 128, 3, 1), (65536, 32, 129, 2), (32769, 64, 5, 17), (65536, 64, 18, 16)]


def whole_weights(n, group, groups, mins, seed, scales=(-1.0, -0.5, 0.25, 0.5, 1.0)):
    """4-bit weights whose scales are powers of two and whose least values are quarters, and their values [n, k] in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda high, shape, t: torch.randint(0, high, shape, generator=g, device="cuda", dtype=t)  # noqa: E731
    codes = draw(256, (n, group * groups // 2), torch.uint8)
    s = torch.tensor(scales, dtype=torch.float16, device="cuda")[draw(len(scales), (n, groups), torch.int64)]
    least = ((draw(33, (n, groups), torch.int64) - 16).double() / 4).to(torch.float16) if mins else None
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(n, groups, group).double()
    w = s.double()[..., None] * c + least.double()[..., None] if mins else s.double()[..., None] * (c - 8)
    return codes, s, least, w.reshape(n, -1)


@pytest.mark.parametrize("act", ["f32", "f16", "bf16", "int8"])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("n,group,groups,m", Q4_SHAPES)
def test_q4_products_of_whole_numbers(ops, act, mins, n, group, groups, m):  # noqa: F811
    """x of whole numbers up to 2 and weights of quarters: every sum is a number of quarters under 2^24 in any order, so the result is exact before its
    one rounding, and every column counts: x has something everywhere, in the last group alone, around the 128th group, in a single column."""
    k = group * groups
    assert 4 * k * 2 * (31 + 4) < 1 << 24                       # |x| <= 2, a code with 16 added <= 31, a least value <= 4, in quarters
    codes, s, least, w = whole_weights(n, group, groups, mins, n + groups)
    g = torch.Generator(device="cuda").manual_seed(m)
    full = torch.randint(-2, 3, (m, k), generator=g, device="cuda").double()
    parts = {"all": slice(0, k), "last": slice(k - group, k), "edge": slice(max(0, min(127 * group, k - 2 * group)), min(k, 129 * group)), "one": slice(k - 1, k)}
    for where, at in parts.items():
        x = torch.zeros_like(full)
        x[:, at] = full[:, at] if where != "one" else full[:, at].abs() + 1
        ref = torch.mm(x, w.t().contiguous())
        if act == "int8":
            for one in (True, False):                          # one scale for a row, or one for every group
                xs = torch.full((m, 1 if one else groups), 0.5, device="cuda")
                y = ops.q4_matvec(codes, s, x.to(torch.int8), mins=least, x_scale=xs)
                assert torch.equal(y.double(), 0.5 * ref), (where, one)
        else:
            y = ops.q4_matvec(codes, s, x.to(ACT[act]), mins=least)
            assert torch.equal(y, ref.float().to(ACT[act])), where
    ops.sync()


@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("n,group,groups,m", Q4_SHAPES)
def test_q4_products_keep_all_of_a_32_bit_x(ops, mins, n, group, groups, m):  # noqa: F811
    """x has three columns of 1 + 2^-10 + 2^-18, one for each of the bf16 that carry it.  A code with 16 added makes that 23 bits, the sum of three with least
    values under 2^6 has 24: exact in any order (but where all three meet in one block), and without the last part off by 2^-18 of a weight."""
    k = group * groups
    codes, s, least, w = whole_weights(n, group, groups, mins, n, scales=(-1.0, 1.0))
    least = None if least is None else least.round()
    if mins:
        c = torch.stack((codes & 15, codes >> 4), -1).reshape(n, groups, group).double()
        w = (s.double()[..., None] * c + least.double()[..., None]).reshape(n, k)
    value = 1 + 2.0 ** -10 + 2.0 ** -18
    x = torch.zeros((m, k), dtype=torch.float64, device="cuda")
    for i in range(m):
        for at in {(3 + 5 * i) % k, k // 2, k - 1 - i % group}:
            x[i, at] = value if i % 2 else -value
    assert bool((x.float().double() == x).all())
    ref = torch.mm(x, w.t().contiguous())
    y = ops.q4_matvec(codes, s, x.float(), mins=least)
    ops.sync()
    # two columns in one block of 32 give codes with 16 added up to 2 * 31 * value < 2^6, 24 bits; all three in one, where there is but one block, up to
    # 3 * 31 * value < 2^7, so each of the nine additions there, the step that takes 24 off and the two into the sums may round by half of 2^-17
    assert float((y.double() - ref).abs().max()) <= (12 * 2.0 ** -18 if k == 32 else 0)


@pytest.mark.parametrize("n,group,groups,m", [(33, 64, 3, 2), (100, 32, 129, 5), (70, 32, 257, 17), (8193, 32, 260, 2), (65536, 32, 129, 2), (16390, 32, 33, 17)])
@pytest.mark.parametrize("mins", [False, True])
def test_q4_error_of_32_bit_rows(ops, mins, n, group, groups, m):  # noqa: F811
    """The root mean square of the error where roundings are independent.  Of a scale's worth, x of spread 1: a block of 32 columns has up to 3 x 32 additions
    (two such blocks, with codes and with ones) whose partial sums are up to 31 sqrt(32) (times 24 for the ones) / 24, so sqrt(2 * 3 k) * 31 * sqrt(32);
    the k / 32 blocks and 2 k / group steps of the sums over them have partial sums of up to (8 + |least| / |scale|) sqrt(k).  Each rounding is under 2^-24 of its partial sum."""
    k = group * groups
    codes, s, least, w = whole_weights(n, group, groups, mins, groups, scales=(-1.0, 1.0))
    x = rnd((m, k), torch.float32, 5).cuda()
    ref = torch.mm(x.double(), w.t().contiguous())
    y = ops.q4_matvec(codes, s, x, mins=least)
    ops.sync()
    rms = float((y.double() - ref).square().mean().sqrt())
    bound = 2.0 ** -24 * (math.sqrt(6 * k) * 31 * math.sqrt(32) + math.sqrt(k / 32 + 2 * k / group) * (16 + 4) * math.sqrt(k) + float(ref.square().mean().sqrt()))
    assert rms <= bound, rms / bound


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
def test_q4_products_of_small_numbers(ops, act):  # noqa: F811
    """x around the least normal number of its type, subnormal ones among them, bit for bit; of 32-bit ones bits under 2^-133 are lost, no more."""
    codes, s, least, w = whole_weights(50, 32, 9, False, 3, scales=(-1.0, 1.0))
    step = {"f32": 2.0 ** -133, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}[act]
    g = torch.Generator(device="cuda").manual_seed(1)
    for big in (3, 100):
        x = torch.randint(-big, big + 1, (4, 288), generator=g, device="cuda").double() * step
        assert bool((x.to(ACT[act]).double() == x).all())
        ref = torch.mm(x, w.t().contiguous())
        y = ops.q4_matvec(codes, s, x.to(ACT[act]))
        ops.sync()
        assert torch.equal(y, ref.float().to(ACT[act])), big
    if act == "f32":
        for e in (-104, -112, -118, -124, -130):
            x = (rnd((4, 288), torch.float32, 7) * 2.0 ** e).cuda()
            ref = torch.mm(x.double(), w.t().contiguous())
            y = ops.q4_matvec(codes, s, x)
            ops.sync()
            # cut off below 2^-133, times a weight of up to 8; the rest as in any product (31 for a code with 16 added, 24 off again: 55)
            bound = 288 * 8 * 2.0 ** -133 + (288 + 16) * 2.0 ** -24 * 55 * x.double().abs().sum(-1, keepdim=True) + 2.0 ** -149
            assert bool(((y.double() - ref).abs() <= bound).all()), e


# ---------------------------------------------------------------------------------------------------------------------
# the operators together
class Recorded(Layer):
    """A layer whose products are all kept: `out` name -> (rows, their scales, result)."""

    def project(self, ops, name, x, x_scale=None):  # noqa: F811
        y = super().project(ops, name, x, x_scale)
        self.out[name] = (x, x_scale, y)
        return y


def check_residual_norm(x, r, w, total, codes, scales, eps, group):
    """bf16 rows to int8, as check_norm bounds them: the sum is one rounding, y has cols / 2 + 12 in 32 bits, a code half a step."""
    s = x.double() + r.double()
    assert bool(((total.double() - s).abs() <= (u(torch.bfloat16) + 2 * U32) * s.abs()).all())
    cols = x.shape[1]
    y = (s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * w.double()).reshape(x.shape[0], -1, group)
    rel = (cols / 2 + 12) * U32
    top, sc = y.abs().amax(-1), scales.double()
    assert bool(((sc - top / 127).abs() <= (rel + 4 * U32) * top / 127).all())
    back = codes.double().reshape(y.shape) * sc[..., None]
    assert bool(((back - y).abs() <= (rel * y.abs() + sc[..., None] * (0.5 + 127 * 4 * U32)) * (1 + 1e-6)).all())


@pytest.mark.parametrize("store", ["same", "e4m3"])
def test_every_stage_of_a_layer(ops, store):  # noqa: F811
    """All four products and both norms of a layer's token steps against 64 bits on the stage's own inputs."""
    lay, B = Recorded(seed=5), 3
    lay.out = {}
    P = Paged(ops, [0, 7, 29], lay.kv, lay.hd, 8, "bf16", store, seed=3, extra_pages=24, width=8)
    used = set(P.table[P.table >= 0].tolist())
    free = iter([p for p in range(P.cache.n_pages) if p not in used])
    table = torch.tensor([[p if p >= 0 else next(free) for p in row] for row in P.table.tolist()], dtype=torch.int32, device="cuda")
    x, res = rnd((B, 256), torch.bfloat16, 1).cuda(), rnd((B, 256), torch.bfloat16, 2).cuda()
    for t in range(6):
        lens, keep = [n + t + 1 for n in P.lens], {}
        d, h2 = lay.step(ops, x, res, P.cache, table, ints(lens), ints([0, 1, 2, 3]), ints([n - 1 for n in lens]), 64, keep)
        ops.sync()
        kk = {n: v.cpu() for n, v in keep.items()}
        check_residual_norm(x.cpu(), res.cpu(), lay.norm[0], kk["h"], kk["c"], kk["s"], 1e-5, 32)
        check_residual_norm(kk["o"], kk["h"], lay.norm[1], kk["h2"], kk["c2"], kk["s2"], 1e-5, 32)
        assert set(lay.out) == {"qkv", "o", "up", "down"}
        for name, (xin, sc, y) in lay.out.items():
            _, _, least, w, s = lay.w[name]
            xv = xin.cpu().double() if sc is None else xin.cpu().double() * sc.cpu().double().repeat_interleave(32, 1)
            ref = xv @ w.t()
            mag = xv.abs() @ (55 * s).t() + (xv.abs() @ least.double().abs().repeat_interleave(32, 1).t() if least is not None else 0)
            assert bool(((y.cpu().double() - ref).abs() <= 1.01 * (mag * (xv.shape[1] + 16) * U32 + u(torch.bfloat16) * ref.abs())).all()), name
        assert torch.equal(kk["f"], torch.nn.functional.silu(lay.out["up"][2]).cpu())
        x, res = d, h2
