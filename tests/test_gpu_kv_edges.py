"""GPU suite of the quantised KV cache at its edges: scores, lists and arguments at the ends of what the
calls take, against the definitions in 64 bits (tests/kv_reference.py)."""
import numpy as np
import pytest
import torch

from tests import kv_reference as R
from tests.test_gpu_kv import attend_case, dev, kv, make, rows_of, verify  # noqa: F401  (kv: a fixture)

pytestmark = pytest.mark.gpu


# ---- scores ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,cache", [("fp16", "fp16"), ("bf16", "bf16")])
@pytest.mark.parametrize("n,per", [(1, 4), (16, 4), (32, 4), (64, 4)])  # tiles of 16, 64, 128, 256 rows
@pytest.mark.parametrize("first,second", [(5, 37), (5, 69), (5, 133)])
@pytest.mark.parametrize("key", [(16344, 2474, 6), (20432, 1862, 9), (65440, 1969, 15), (65504, 308, 16)])
def test_scores_past_two_to_the_25(kv, dtype, cache, n, per, first, second, key):
    """Two tokens with scores of 2.7e8 to 1.1e9, exact in 32 bits and 32 to 128 apart, the larger one later:
    the weights' exponents are off by up to a step of such a score, but a weight stays finite.  Both tokens hold
    the same values, so whatever their weights are the outputs are those values."""
    batch, heads, dim, length, page = 64, 32, 64, 192, 64
    dt = torch.float16 if dtype == "fp16" else torch.bfloat16
    c = make(kv, cache, 3 + batch, page, heads, dim)
    c.k.fill_(0)
    g = torch.Generator(device="cuda").manual_seed(3)
    c.v.copy_(torch.randn(c.v.shape, generator=g, device="cuda"))
    a, b, m = key
    # (the drafts' own tokens are in a page of each sequence's own; keys of zeros: weights of zero)
    for at, row in ((first, (a, b, 0)), (second, (a, b, m))):
        c.k[at // page, at % page, :, :3] = torch.tensor(row, dtype=torch.float32, device="cuda").to(dt)
    c.v[second // page, second % page] = c.v[first // page, first % page]
    want = c.v[first // page, first % page].float()  # [heads, dim]
    table = dev(np.concatenate([np.tile(np.arange(3), (batch, 1)), 3 + np.arange(batch)[:, None]], 1).astype(np.int32))
    kv_len = dev(np.full(batch, length + n, np.int32))
    cu = dev((np.arange(batch + 1) * n).astype(np.int32))
    q = torch.zeros(batch * n, heads * per, dim, device="cuda", dtype=dt)
    q[..., :3] = torch.tensor([16384.0, 64.0, 8.0], device="cuda").to(dt)
    got, lse = c.attend(q, table, kv_len, cu, max_q=n, scale=128 ** -0.5, lse=True)
    c.ctx.sync()
    u = torch.finfo(dt).eps / 2
    want = want.repeat_interleave(per, 0)
    # sums of two products each in 32 bits (the other weights are zero) and a quotient, then the type's rounding
    assert ((got.float() - want).abs() <= want.abs() * (u + 8 * 2.0 ** -24) * 1.01).all()
    assert torch.isfinite(lse).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("n,per", [(1, 4), (16, 4), (32, 4), (64, 4)])
@pytest.mark.parametrize("below", [14, 20, 22])
def test_many_small_weights(kv, fmt, dtype, n, per, below):
    """One token, and 60000 whose weights are 2^-below of its own: in fp16 they are near and below its smallest
    normal number, and carry a part of the outputs that is seen."""
    heads, dim, length, page = 1, 64, 60000, 64
    dt = torch.float16 if dtype == "fp16" else torch.bfloat16
    pages = -(-(length + n) // page)
    c = make(kv, fmt, pages, page, heads, dim, 64)
    c.k.fill_(0)
    c.k_scale.fill_(127)
    c.v_scale.fill_(127)
    c.v.fill_(0x38 if fmt == "e4m3" else 0x22)  # ones
    c.k[0, 7, 0, 0] = 0x38 if fmt == "e4m3" else 0x02  # 1.0 in the first element
    c.v[0, 7] = 0x40 if fmt == "e4m3" else 0x44  # twos
    q = torch.zeros(n, heads * per, dim, device="cuda", dtype=dt)
    q[..., 0] = 1.0
    scale = below * float(np.log(2.0))
    got, lse = c.attend(q, dev(np.arange(pages, dtype=np.int32)[None]), dev(np.array([length + n], np.int32)),
                        dev(np.array([0, n], np.int32)), max_q=n, scale=scale, lse=True)
    c.ctx.sync()
    seen = length + 1 + np.arange(n)  # tokens of each row
    p = 2.0 ** -float(below)
    small = (seen - 1) * p
    want = torch.from_numpy((2.0 + small) / (1.0 + small))[:, None, None]
    u = torch.finfo(dt).eps / 2
    # the reference's bound with its terms for this case: weights rounded (u, twice), their exponents, sums of
    # 60000 terms in 32 bits (twice), and what falls under fp16's range
    rel = 2 * u + 2 * ((dim + 8) * 2.0 ** -24 * scale * 1.5 + 2.0 ** -20) + 2 * length * 2.0 ** -24 + length * 2.0 ** -31
    # an error of a weight moves the quotient only as far as the values differ (by 1 of at most 2): the part of it
    # that all weights share cancels
    assert ((got.cpu().double() - want).abs() <= u * want + 1.01 * rel * want).all()
    # (and closer: the small weights are all alike, so their sums are off by one relative error in all, at most a
    # rounding of a weight and the sums': the outputs see that of the small part alone)
    part = torch.from_numpy(small / (1.0 + small) ** 2)[:, None, None]
    step = 2.0 ** -24 / 2.0 ** (7 - below) if dtype == "fp16" and below > 21 else 2 * u  # half a subnormal's step: 2^-25
    near = u * want + part * (2 * step + 4 * u) + 2 * length * 2.0 ** -24 * 2
    assert ((got.cpu().double() - want).abs() <= near).all()
    ref = torch.from_numpy(scale + np.log1p(small))[:, None]
    assert ((lse.cpu().double() - ref).abs() <= length * 2.0 ** -24 + 2.0 ** -19 + 2.0 ** -21 * ref).all()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2", "e2m1"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,per", [(1, 3), (20, 3), (50, 4)])
def test_scale_bytes_at_their_ends(kv, fmt, dtype, n, per):
    """Scale bytes of 0 and 255 among a caller's own: 2^-127, and NaN that reaches the rows that see it alone."""
    f, dim = {"e4m3": R.E4M3, "e5m2": R.E5M2, "e2m1": R.E2M1}[fmt], 64
    rng = np.random.default_rng(5)
    past, page = 70, 16
    length = past + n
    pages = -(-length // page)
    c = make(kv, fmt, pages, page, 1, dim, 32)
    table, kv_len, cu = np.arange(pages, dtype=np.int32)[None], np.array([length], np.int32), np.array([0, n], np.int32)
    x = rows_of(rng, length, 1, dim, dtype)
    full = dev(np.array([0, length], np.int32))
    c.write(x.cuda(), x.cuda(), dev(table), dev(kv_len), full)
    c.ctx.sync()
    c.k_scale[0, 0, 1, 3] = 0      # a token of the past with tiny keys
    c.v_scale[1, 0, 0, 5] = 0      # ... and with tiny values
    c.v_scale[2, 0, 1, 1] = 1
    last = length - 1              # the last row alone sees NaN values
    c.v_scale[last // page, 0, 1, last % page] = 255
    back = c.read(dev(table), dev(kv_len), full, rows=length, dtype=torch.float32)
    q = rows_of(rng, n, per, dim, dtype, 0.7)
    got, lse = c.attend(q.cuda(), dev(table), dev(kv_len), dev(cu), max_q=n, lse=True)
    c.ctx.sync()
    k, v = R.pool_values(c.k, c.k_scale, f), R.pool_values(c.v, c.v_scale, f)
    for t, pool in zip(back, (k, v)):
        want = torch.from_numpy(pool.reshape(-1, 1, dim)[:length]).float()
        assert torch.equal(t.cpu().nan_to_num(nan=12345.0), want.nan_to_num(nan=12345.0))
    out, ref, weight = R.attend(q.double().numpy(), k, v, table, kv_len, cu, None, dim ** -0.5)
    got = got.cpu().double().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(out)) and np.isnan(out[-1, :, 32:]).all() and not np.isnan(out[:-1]).any()
    fin = np.isfinite(out)
    dt = torch.float16 if dtype == "fp16" else torch.bfloat16
    tol = R.tolerance(np.where(fin, out, 0), np.where(fin, weight, 0), q.double().numpy(), float(np.abs(k[np.isfinite(k)]).max()),
                      length, dim ** -0.5, dt)
    assert (np.abs(np.where(fin, got, 0) - np.where(fin, out, 0)) <= tol).all()
    assert np.isfinite(lse.cpu().numpy()).all()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2", "e2m1"])
@pytest.mark.parametrize("n,per", [(1, 3), (20, 3), (50, 4)])
def test_fp16_queries_take_values_as_fp16_reads_them(kv, fmt, n, per):
    """Values of a past token and of a draft beyond 65504 are infinite for fp16 queries, as hf_kv_read gives them,
    and reach the rows that see them."""
    f, dim, past, page = {"e4m3": R.E4M3, "e5m2": R.E5M2, "e2m1": R.E2M1}[fmt], 64, 70, 16
    length = past + n
    pages = -(-length // page)
    c = make(kv, fmt, pages, page, 1, dim, 32)
    rng = np.random.default_rng(8)
    table, kv_len, cu = np.arange(pages, dtype=np.int32)[None], np.array([length], np.int32), np.array([0, n], np.int32)
    x = rows_of(rng, length, 1, dim, "fp16").cuda()
    full = dev(np.array([0, length], np.int32))
    c.write(x, x, dev(table), dev(kv_len), full)
    c.ctx.sync()
    seen_by_all, group = 9, {"e4m3": 136, "e5m2": 129, "e2m1": 142}[fmt]  # a part of the values passes 65504
    c.v_scale[0, 0, 0, seen_by_all] = group
    draft = length - 1
    c.v_scale[draft // page, 0, 1, draft % page] = group
    read = c.read(dev(table), dev(kv_len), full, rows=length, dtype=torch.float16)[1]
    q = rows_of(rng, n, per, dim, "fp16", 0.7)
    got, lse = c.attend(q.cuda(), dev(table), dev(kv_len), dev(cu), max_q=n, lse=True)
    c.ctx.sync()
    k, v = R.pool_values(c.k, c.k_scale, f), R.pool_values(c.v, c.v_scale, f)
    flat = torch.from_numpy(v.reshape(-1, 1, dim)[:length]).to(torch.float16)
    assert torch.equal(read.cpu(), flat)
    assert torch.isinf(flat[seen_by_all, 0, :32]).any() and torch.isinf(flat[draft, 0, 32:]).any()
    v16 = np.zeros_like(v)
    v16.reshape(-1, 1, dim)[:length] = flat.double().numpy()
    out, ref, weight = R.attend(q.double().numpy(), k, v16, table, kv_len, cu, None, dim ** -0.5)
    got = got.cpu().double().numpy()
    fin = np.isfinite(out)
    assert np.array_equal(got[~fin], out[~fin]) and np.isfinite(got[fin]).all()
    tol = R.tolerance(np.where(fin, out, 0), np.where(fin, weight, 0), q.double().numpy(), float(np.nanmax(np.abs(k[np.isfinite(k)]))),
                      length, dim ** -0.5, torch.float16)
    assert (np.abs(np.where(fin, got, 0) - np.where(fin, out, 0)) <= tol).all()


# ---- lists -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("past", [0, 1, 20])
@pytest.mark.parametrize("path", [[-2, -1], [-5, -3], [-1, 0], [-2 ** 31, -2 ** 31 + 1], [-3, 2], [0, 2 ** 31 - 1], [-2 ** 31, 3]])
def test_paths_below_zero_are_reported_and_move_nothing(kv, hf, past, path):
    from huffman_amd import HuffhipError
    ctx = hf.Context()
    c = make(kv, "e4m3", 4, 16, 2, 64, 32, ctx=ctx)
    g = torch.Generator(device="cuda").manual_seed(2)
    for pool in (c.k, c.v):
        pool.copy_(torch.randint(0, 0x70, pool.shape, generator=g, device="cuda", dtype=torch.uint8))
    before = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    table, cu = dev(np.array([[3, 1], [2, 0]], np.int32)), dev(np.array([0, 4, 8], np.int32))
    kv_len = np.array([past + 4, past + 4], np.int32)
    torch.cuda.synchronize()
    new_len = c.keep(table, dev(kv_len), cu, dev(np.array([path, [0, 1]], np.int32)), dev(np.array([2, 2], np.int32)))
    with pytest.raises(HuffhipError):
        ctx.sync()
    assert new_len.tolist() == [past + 4, past + 2]  # (the other sequence's path stays where it is)
    for t, was in zip((c.k, c.v, c.k_scale, c.v_scale), before):
        assert torch.equal(t, was)


@pytest.mark.parametrize("call", ["write", "read"])
@pytest.mark.parametrize("batch", [3, 1500])
@pytest.mark.parametrize("what", ["falls", "leaves", "negative length", "long length", "fewer tokens"])
def test_every_list_that_does_not_fit_is_reported(kv, hf, call, batch, what):
    """Offsets that fall although the sequence behind them is long enough for the rows it then claims, offsets
    that leave the rows, and lengths of sequences without rows, which no row of the call leads to."""
    from huffman_amd import HuffhipError
    ctx = hf.Context()
    page, width = 16, 8
    c = make(kv, "e4m3", batch * width, page, 1, 64, 64, ctx=ctx)
    table = np.arange(batch * width, dtype=np.int32).reshape(batch, width)
    rows = 9
    cu = np.full(batch + 1, rows, np.int32)
    cu[:3] = [0, 6, 6]  # 6 rows, none, 3, none ...
    kv_len = np.full(batch, 100, np.int32)
    x = torch.ones(rows, 1, 64, device="cuda", dtype=torch.bfloat16)
    out = (x.clone(), x.clone())
    torch.cuda.synchronize()

    def run(kv_len, cu):
        if call == "write":
            c.write(x, x, dev(table), dev(kv_len), dev(cu))
        else:
            c.read(dev(table), dev(kv_len), dev(cu), out=out)
        torch.cuda.synchronize()

    run(kv_len, cu)
    ctx.sync()  # as it should be: nothing to report
    bad_len, bad_cu = kv_len.copy(), cu.copy()
    if what == "falls":
        bad_cu[2] = 3
    elif what == "leaves":
        bad_cu[3:] = rows + 4
        bad_cu[2] = rows  # (the third sequence's rows all lie behind the tensors)
    elif what == "negative length":
        bad_len[1] = -1
    elif what == "long length":
        bad_len[1] = page * width + 1
    else:
        bad_cu[1:] = rows
        bad_cu[0] = rows - 1
        bad_len[0] = 0
    run(bad_len, bad_cu)
    with pytest.raises(HuffhipError):
        ctx.sync()
    run(kv_len, cu)
    ctx.sync()


# ---- arguments -------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape,dim", [((1, 16, 8, 128), 1), ((1, 16, 8, 128), 2), ((4, 16, 1, 128), 0), ((4, 16, 1, 128), 1),
                                       ((4, 16, 8, 128), 0), ((4, 16, 8, 128), 1), ((4, 16, 8, 128), 2)])
def test_pools_whose_rows_lie_on_one_another_are_refused(kv, shape, dim):
    """Expanded pools, also where another dimension is one and its stride is made up."""
    from huffman_amd import HuffhipError
    pages, page, heads, width = shape
    pools = [torch.zeros(shape, dtype=torch.uint8, device="cuda").narrow(dim, 0, 1).expand(shape) for _ in range(2)]
    scales = [torch.full((pages, heads, 1, page), 127, dtype=torch.uint8, device="cuda") for _ in range(2)]
    c = kv.KvCache(*pools, *scales)
    t, l = dev(np.zeros((1, 1), np.int32)), dev(np.full(1, 16, np.int32))
    x = torch.ones(1, heads, width, device="cuda", dtype=torch.bfloat16)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    for call in (lambda: c.write(x, x, t, l), lambda: c.read(t, l), lambda: c.attend(x, t, l),
                 lambda: c.keep(t, l, None, zero[None], zero)):
        with pytest.raises(HuffhipError):
            call()
    c.ctx.sync()


def test_new_lengths_in_memory_that_the_call_reads_are_refused(kv):
    """Every list of the call, whole or in part, may be in use when the first length is written; what lies
    between the rows of a wider table or path is not."""
    from huffman_amd import HuffhipError
    c = make(kv, "e4m3", 4, 16, 2, 64, 32)
    buf = torch.zeros(64, dtype=torch.int32, device="cuda")
    cu, length, kept = buf[0:3], buf[3:5], buf[5:7]
    wide_path, wide_table = buf[16:32].view(2, 8), buf[32:48].view(2, 8)
    path, table = wide_path[:, :3], wide_table[:, :2]
    cu.copy_(dev(np.array([0, 3, 6], np.int32)))
    length.copy_(dev(np.array([9, 20], np.int32)))
    kept.copy_(dev(np.array([2, 1], np.int32)))
    path.copy_(dev(np.array([[0, 2, 9], [1, 0, 0]], np.int32)))
    table.copy_(dev(np.array([[0, 1], [2, 3]], np.int32)))
    torch.cuda.synchronize()
    before = buf.clone()
    for lo in (0, 1, 2, 3, 4, 5, 6, 15, 16, 17, 18, 23, 24, 26, 31, 32, 33, 39, 40, 41):
        with pytest.raises(HuffhipError):
            c.keep(table, length, cu, path, kept, new_len=buf[lo:lo + 2])
    c.ctx.sync()
    assert torch.equal(buf, before)
    for lo in (7, 14, 19, 22, 27, 29, 34, 38, 42, 48):
        assert c.keep(table, length, cu, path, kept, new_len=buf[lo:lo + 2]).tolist() == [8, 18]
    c.ctx.sync()


def test_a_scale_whose_logarithmic_form_overflows_is_refused(kv):
    from huffman_amd import HuffhipError
    c = make(kv, "e4m3", 4, 16, 2, 64, 32)
    c.k.fill_(0)
    c.v.fill_(0x38)
    t, l = dev(np.zeros((1, 1), np.int32)), dev(np.ones(1, np.int32))
    q = torch.zeros(1, 4, 64, device="cuda", dtype=torch.bfloat16)
    for scale in (2.4e38, 3.0e38, 3.4e38):
        with pytest.raises(HuffhipError):
            c.attend(q, t, l, scale=scale)
    for scale in (2.3e38, 1e-38, 1e-44):  # scores of zero: ones
        assert (c.attend(q, t, l, scale=scale) == 1).all()
    c.ctx.sync()


def test_a_refused_call_leaves_the_next_one_alone(kv):
    """A table whose rows lie on one another is refused; the same shape in a table of its own is not."""
    from huffman_amd import HuffhipError
    c = make(kv, "e4m3", 64, 16, 2, 64, 32)
    c.k.fill_(0)
    c.v.fill_(0x38)
    row, l = dev(np.arange(32, dtype=np.int32)[None]), dev(np.full(2, 500, np.int32))
    q = torch.zeros(2, 4, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(HuffhipError):
        c.attend(q, row.expand(2, 32), l)
    assert (c.attend(q, row.repeat(2, 1), l) == 1).all()
    c.ctx.sync()


def test_lists_of_one_entry_may_have_any_stride(kv):
    c = make(kv, "e4m3", 4, 16, 2, 64, 32)
    x = torch.ones(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    state = dev(np.array([[5, 2, 1, 0]], np.int32))  # one sequence's length, page, accepted drafts and path
    length, page, kept, path = state[:, 0], state[:, 1:2], state[:, 2], state[:, 3:4]
    assert length.stride() == (4,)
    c.write(x, x, page, length)
    assert (c.read(page, length)[0] == 1).all()
    assert (c.attend(x.repeat(1, 2, 1), page, length).shape == (1, 4, 64))
    assert c.keep(page, length, None, path, kept).tolist() == [5]
    assert c.keep(page.t(), length, None, path.t(), kept).tolist() == [5]
    c.ctx.sync()


def test_tensors_that_need_gradients_are_refused(kv):
    """No call records what a backward pass needs."""
    c = make(kv, "e4m3", 4, 16, 2, 64, 32)
    t, l = dev(np.zeros((1, 1), np.int32)), dev(np.ones(1, np.int32))
    x = torch.ones(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    q = torch.ones(1, 4, 64, device="cuda", dtype=torch.bfloat16)
    need = lambda a: a.clone().requires_grad_()  # noqa: E731
    for call in (lambda: c.write(need(x), x, t, l), lambda: c.write(x, need(x), t, l), lambda: c.attend(need(q), t, l),
                 lambda: c.attend(need(q) * 1, t, l), lambda: c.attend(q, t, l, out=need(q)),
                 lambda: c.read(t, l, out=(x.clone(), need(x)))):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad():
            call()
    with torch.inference_mode():
        c.attend(need(q), t, l)
    c.ctx.sync()


def test_outputs_that_lie_on_one_another_are_refused(kv):
    """Heads of a row on the rows behind it; layouts whose rows stay apart in any order are taken."""
    from huffman_amd import HuffhipError
    c = make(kv, "e4m3", 4, 16, 3, 64, 32)
    g = torch.Generator(device="cuda").manual_seed(4)
    for pool in (c.k, c.v):
        pool.copy_(torch.randint(0, 0x70, pool.shape, generator=g, device="cuda", dtype=torch.uint8))
    t, l, cu = dev(np.array([[2, 1]], np.int32)), dev(np.full(1, 20, np.int32)), dev(np.array([0, 2], np.int32))
    q = torch.randn(2, 3, 64, generator=g, device="cuda").bfloat16()
    want, rows = c.attend(q, t, l, cu, max_q=2), c.read(t, l, cu, rows=2)
    flat = lambda: torch.zeros(2048, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    for strides in ((64, 64), (128, 64), (96, 64), (192, 96)):
        out = flat().as_strided((2, 3, 64), strides + (1,))
        good = flat()[:384].view(2, 3, 64)
        for call in (lambda: c.attend(q, t, l, cu, max_q=2, out=out), lambda: c.read(t, l, cu, out=(out, good)),
                     lambda: c.read(t, l, cu, out=(good, out))):
            with pytest.raises(HuffhipError):
                call()
    for strides in ((192, 64), (64, 192), (64, 128), (200, 64), (192, 128), (1024, 72)):
        out, other = (flat().as_strided((2, 3, 64), strides + (1,)) for _ in range(2))
        assert torch.equal(c.attend(q, t, l, cu, max_q=2, out=out), want)
        got = c.read(t, l, cu, out=(out, other))
        assert torch.equal(got[0], rows[0]) and torch.equal(got[1], rows[1])
    c.ctx.sync()


@pytest.mark.parametrize("n,per,past", [(1, 4, 3000), (5, 4, 20), (33, 4, 40), (70, 4, 40)])
def test_outputs_over_what_the_call_reads_or_writes(kv, n, per, past):
    """Outputs over the queries themselves, row for row, are as anywhere else; over other rows of them, or keys
    over values, they are refused."""
    from huffman_amd import HuffhipError
    c, f, q, table, kv_len, cu, _ = attend_case(kv, "e4m3", "bf16", [n, n], [past, 7], 16, 2, per, 64, 64, "thd", None, 3)
    lists = dev(table), dev(kv_len), dev(cu)
    q = q.cuda()
    want = c.attend(q, *lists, max_q=n)
    buf = torch.zeros(2 * n + 1, 2 * per, 64, device="cuda", dtype=torch.bfloat16)
    for lo in (0, 1):
        same = buf[lo:lo + 2 * n]
        same.copy_(q)
        assert c.attend(same, *lists, max_q=n, out=same) is same and torch.equal(same, want)
    for a, b in ((0, 1), (1, 0)):
        with pytest.raises(HuffhipError):
            c.attend(buf[a:a + 2 * n], *lists, max_q=n, out=buf[b:b + 2 * n])
    flat = torch.zeros(2 * n * 2 * per * 64, device="cuda", dtype=torch.bfloat16)
    turned = flat.view(2 * per, 2 * n, 64).transpose(0, 1)  # the same memory, heads in front
    turned.copy_(q)
    with pytest.raises(HuffhipError):
        c.attend(turned, *lists, max_q=n, out=flat.view(q.shape))
    assert torch.equal(c.attend(turned, *lists, max_q=n, out=turned), want)
    rows = torch.zeros(2 * n + 1, 3, 64, device="cuda", dtype=torch.bfloat16)
    for k, v in ((rows[1:, :2], rows[1:, :2]), (rows[1:, :2], rows[1:, 1:]), (rows[1:, 1:], rows[1:, :2]),
                 (rows[1:, :2], rows[:-1, :2]) if n > 1 else (rows[1:, :2], rows[1:, :2])):
        with pytest.raises(HuffhipError):
            c.read(*lists, out=(k, v))
    good = c.read(*lists, rows=2 * n)
    wide = torch.zeros(2 * n, 4, 64, device="cuda", dtype=torch.bfloat16)
    got = c.read(*lists, out=(wide[:, 2:], wide[:, :2]))
    assert torch.equal(got[0], good[0]) and torch.equal(got[1], good[1])
    got = c.read(*lists, out=(wide[:, ::2], wide[:, 1::2]))
    assert torch.equal(got[0], good[0]) and torch.equal(got[1], good[1])
    c.ctx.sync()


# ---- streams ---------------------------------------------------------------------------------------
def test_tensors_dropped_before_another_stream_has_used_them(kv, hf):
    """Every tensor of a call on a context's own stream, which is busy, is dropped right after the call and
    its memory asked for again: the call works on what it was given."""
    side = torch.cuda.Stream()
    ctx = hf.Context(stream=side)
    heads, dim, n = 4, 128, 512
    c = make(kv, "bf16", 64, 16, heads, dim, ctx=ctx)
    a = torch.randn(4096, 4096, device="cuda")
    k, v = (torch.randn(n, heads, dim, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(n, heads, dim, device="cuda").bfloat16()
    lists = [np.arange(32, dtype=np.int32)[None], np.array([n], np.int32), np.array([0, n], np.int32)]
    steps = [np.arange(0, n, 2, dtype=np.int32)[None], np.array([n // 2], np.int32)]

    def spoil(sizes):
        return [torch.full((s,), 0x55, dtype=torch.uint8, device="cuda") for s in sizes for _ in range(3)]

    def run(early):
        got = []
        for i in range(4):
            given = [t.clone() for t in ([k, v] if i == 0 else [q] if i == 2 else [])]
            given += [dev(x) for x in lists + (steps if i == 3 else [])]
            torch.cuda.synchronize()
            if early:
                with torch.cuda.stream(side):
                    for _ in range(8):
                        torch.mm(a, a)
            if i == 0:
                c.write(*given)
            elif i == 1:
                got += c.read(*given, rows=n)
            elif i == 2:
                got += c.attend(*given, max_q=n, lse=True)
            else:
                got.append(c.keep(*given))
            sizes = [t.numel() * t.element_size() for t in given]
            if early:
                del given
                spoil(sizes)
            torch.cuda.synchronize()
        return got + [c.k.clone(), c.v.clone()]

    want = run(False)
    got = run(True)
    ctx.sync()
    for x, y in zip(want, got):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


# ---- shapes ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("fmt", ["bf16", "fp16", "e4m3", "e5m2", "e2m1"])
@pytest.mark.parametrize("dim,heads,per,new,past,mask", [
    (160, 2, 4, [1, 1, 1], [0, 40, 700], None), (192, 1, 8, [1], [2100], None), (160, 1, 2, [70], [33], None),
    (192, 2, 3, [9, 0, 31], [5, 0, 100], "tree"), (64, 1, 100, [3], [50], None), (32, 3, 1, [200], [0], None),
    (128, 1, 300, [1, 1], [90, 10], None)])
def test_attend_other_shapes(kv, fmt, dtype, dim, heads, per, new, past, mask):
    if fmt in ("bf16", "fp16") and fmt != dtype:
        pytest.skip("a 16-bit cache takes queries of its own type")
    c, f, q, table, kv_len, cu, m = attend_case(kv, fmt, dtype, new, past, 16, heads, per, dim, 32, "thd", mask, 17)
    one = max(new) == 1
    got, lse = c.attend(q.cuda(), dev(table), dev(kv_len), None if one else dev(cu), max_q=max(new),
                        mask=None if m is None else dev(m.view(np.int32)), lse=True)
    c.ctx.sync()
    verify(c, f, q, table, kv_len, cu, m, got, lse, dim ** -0.5, dtype)


@pytest.mark.parametrize("batch", [129, 1025, 4100])
def test_attend_many_sequences_in_large_tiles(kv, batch):
    """More sequences than one pass of the cut takes, most of them of no row or one, a few of up to 40: tiles of
    64 and 256 rows."""
    rng = np.random.default_rng(batch)
    new = rng.integers(0, 2, batch)
    new[rng.integers(0, batch, 20)] = rng.integers(2, 41, 20)
    new[batch - 1] = 40
    past = rng.integers(0, 40, batch)
    past[[batch // 3, batch - 1]] = 3000, 1500  # these are cut into ranges
    for per in (1, 5):
        c, f, q, table, kv_len, cu, _ = attend_case(kv, "e4m3", "bf16", [int(n) for n in new], [int(p) for p in past], 16, 1,
                                                    per, 64, 64, "thd", None, 1)
        got, lse = c.attend(q.cuda(), dev(table), dev(kv_len), dev(cu), max_q=40, lse=True)
        c.ctx.sync()
        verify(c, f, q, table, kv_len, cu, None, got, lse, 64 ** -0.5, "bf16")


@pytest.mark.parametrize("n,per", [(16, 4), (32, 4), (64, 4)])
def test_large_tiles_long_and_past_four_gigabytes(kv, n, per):
    """Tiles of 64, 128 and 256 rows on 20000 tokens in the last pages of a pool of more than 2^32 bytes: bit for
    bit what a dense small pool gives."""
    pages, page, heads, dim = 35000, 64, 16, 128
    if torch.cuda.mem_get_info()[0] < 12e9:
        pytest.skip("needs 12 GB")
    c = kv.KvCache.empty(pages, page, heads, dim, R.E4M3, 128)
    length = 20000 + n
    need = -(-length // page)
    small = kv.KvCache.empty(need, page, heads, dim, R.E4M3, 128)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(length, heads, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(n, heads * per, dim, generator=g, device="cuda").bfloat16()
    far = (pages - 1 - np.random.default_rng(2).permutation(need)).astype(np.int32)[None]
    near = np.arange(need, dtype=np.int32)[None]
    l, cu, full = dev(np.array([length], np.int32)), dev(np.array([0, n], np.int32)), dev(np.array([0, length], np.int32))
    got = []
    for cache, table in ((c, dev(far)), (small, dev(near))):
        cache.write(k, v, table, l, full)
        got.append(cache.attend(q, table, l, cu, max_q=n, lse=True))
    c.ctx.sync()
    assert torch.equal(got[0][0].view(torch.int16), got[1][0].view(torch.int16)) and torch.equal(got[0][1], got[1][1])
    # and one head of it against the definition
    back = small.read(dev(near), l, full, rows=length, dtype=torch.float32)
    small.ctx.sync()
    kk, vv = (t[:, 3].cpu().double().numpy() for t in back)
    qq = q[:, 3 * per + 1].cpu().double().numpy()
    s = qq @ kk.T * dim ** -0.5
    s[np.arange(length)[None] > 20000 + np.arange(n)[:, None]] = -np.inf
    p = np.exp(s - s.max(-1, keepdims=True))
    z = p.sum(-1, keepdims=True)
    out, weight = p @ vv / z, p @ np.abs(vv) / z
    tol = R.tolerance(out, weight, qq, float(np.abs(kk).max()), length, dim ** -0.5, torch.bfloat16)
    assert (np.abs(got[0][0][:, 3 * per + 1].cpu().double().numpy() - out) <= tol).all()


@pytest.mark.parametrize("heads,dim,group", [(1024, 32, 32), (1024, 256, 32), (1000, 224, 32), (513, 160, 32)])
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1", "bf16"])
def test_as_many_heads_as_there_may_be(kv, fmt, heads, dim, group):
    """Rows of up to 32768 pieces, dealt to threads by a multiplication: written, read, kept and attended to."""
    new, past, page = [3, 0, 2], [0, 4, 9], 8
    c, f, q, table, kv_len, cu, _ = attend_case(kv, fmt, "bf16", new, past, page, heads, 1, dim, group, "thd", None, 2)
    lists = dev(table), dev(kv_len), dev(cu)
    x = rows_of(np.random.default_rng(3), 5, heads, dim, "bf16")
    c.write(x.cuda(), (x * 2).cuda(), *lists)
    got = c.read(*lists, rows=5)
    c.ctx.sync()
    if fmt == "bf16":
        want = x.double()
    else:
        want = torch.from_numpy(R.dequantise(*R.quantise(x.double().numpy(), f, group), f, group))
    assert torch.equal(got[0].cpu(), want.bfloat16()) and torch.equal(got[1].cpu(), (2 * want).bfloat16())
    out, lse = c.attend(q.cuda(), *lists, max_q=3, lse=True)
    c.ctx.sync()
    verify(c, f, q, table, kv_len, cu, None, out, lse, dim ** -0.5, "bf16")
    new_len = c.keep(*lists, dev(np.array([[1, 2], [0, 0], [1, 0]], np.int32)), dev(np.array([2, 0, 1], np.int32)))
    assert new_len.tolist() == [2, 4, 10]
    after = c.read(*lists, rows=5)
    for a, b in zip(got, after):
        assert torch.equal(b[[0, 1, 3]], a[[1, 2, 4]]) and torch.equal(b[[2, 4]], a[[2, 4]])
    c.ctx.sync()
