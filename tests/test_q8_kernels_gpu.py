"""The 8-bit cache: written, read back and attended over, against 64-bit plain forms."""
import numpy as np
import pytest
import torch

import plain_q8 as plain
from minfer_b200.kernels import api as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE = 64
FORMATS = pytest.mark.parametrize("fmt", plain.FORMATS, ids=["e4m3", "int8"])


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def status_word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def make_table(ends, ring, rng, spare=2):
    """(table as lists, pages): every row's pages in a random order, -1 behind them."""
    need = [-(-(min(e, ring) if ring else e) // PAGE) for e in ends]
    total = sum(need) + spare
    order = rng.permutation(total).tolist()
    width = max(1, max(need))
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return table, total


def make_pages(table, n_pages, ends, ring, kv, dim, fmt, gen, spread=0.0, junk=True):
    """Pages whose visible places hold random vectors; every other place holds what a use before left:
    codes of any pattern, scales of NaN.  ``spread``: scales differ by up to 2^+-spread."""
    shape = (n_pages, kv, PAGE, dim)
    pages = []
    for _ in range(2):
        x = torch.randn(shape, generator=gen)
        x = x * torch.exp2((torch.rand(shape[:3], generator=gen) * 2 - 1) * spread).unsqueeze(-1)
        pages.append(plain.quantise(x, fmt))
    (k, ks), (v, vs) = pages
    if junk:
        held = torch.zeros(n_pages, PAGE, dtype=torch.bool)
        for b, end in enumerate(ends):
            for p in range(max(0, end - ring) if ring else 0, end):
                place = p % ring if ring else p
                held[table[b][place // PAGE], place % PAGE] = True
        gone = ~held.unsqueeze(1).expand(n_pages, kv, PAGE)
        for code, scale in ((k, ks), (v, vs)):
            code.view(torch.uint8)[gone] = 0x7f
            scale[gone] = float("nan")
    return K.Q8Pages(k.to(DEV), v.to(DEV), ks.to(DEV), vs.to(DEV))


def run_attention(q, pages, cu, ends, table, ring, heads, kv, dim, window, scale, status=None, longest=None, max_end=None):
    out = torch.full_like(q, float("nan"))
    st = status if status is not None else status_word()
    longest = longest if longest is not None else max(1, int(np.diff(cu).max()))
    K.attention_paged_q8(q, pages, ints(cu), ints(ends), ints(table), len(table[0]), ring, out, longest,
                         max_end if max_end is not None else max(1, max(ends)), heads, kv, dim, window, scale, st)
    torch.cuda.synchronize()
    if status is None:
        assert int(st.item()) == 0
    return out


SHAPES = [(28, 4, 128), (14, 2, 64), (4, 4, 64), (5, 1, 128), (20, 1, 64), (6, 2, 96), (4, 1, 16), (2, 1, 256)]
# (new tokens, positions before them) of every row
ROWS = {
    "one": [(1, 0)],
    "borders": [(1, 62), (1, 63), (1, 64), (1, 15), (1, 16), (1, 191)],
    "long-one": [(1, 1500), (1, 3)],
    "few": [(5, 130), (2, 0), (3, 61), (1, 700)],
    "whole": [(70, 0), (33, 5), (64, 64)],
}


@FORMATS
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows", ROWS, ids=list(ROWS))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention(shape, rows, dtype, fmt):
    heads, kv, dim = shape
    gen, rng = torch.Generator().manual_seed(7), np.random.RandomState(3)
    new, past = zip(*ROWS[rows])
    ends = [n + p for n, p in zip(new, past)]
    cu = [0] + np.cumsum(new).tolist()
    table, n_pages = make_table(ends, 0, rng)
    pages = make_pages(table, n_pages, ends, 0, kv, dim, fmt, gen)
    q = (torch.randn(cu[-1], heads, dim, generator=gen) * 1.5).to(dtype).to(DEV)
    scale = dim ** -0.5
    got = run_attention(q, pages, cu, ends, table, 0, heads, kv, dim, 0, scale)
    want, *sizes = plain.attention(q, pages, cu, ends, table, 0, heads, kv, 0, scale)
    tol = plain.attention_tolerance(want, *sizes, dtype, dim, fmt)
    assert ((got.double().cpu() - want).abs() <= tol).all(), float(((got.double().cpu() - want).abs() / tol).max())


@FORMATS
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", [(14, 2, 64), (8, 2, 128), (4, 2, 32)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("window,rows", [(1, [(1, 0), (1, 100)]), (40, [(1, 39), (3, 700), (5, 0)]),
                                         (64, [(1, 63), (1, 64), (4, 126)]), (200, [(9, 500), (1, 90), (2, 199)])])
def test_attention_with_a_window_over_a_ring(window, rows, shape, dtype, fmt):
    heads, kv, dim = shape
    gen, rng = torch.Generator().manual_seed(11), np.random.RandomState(5)
    new, past = zip(*rows)
    ends = [n + p for n, p in zip(new, past)]
    cu = [0] + np.cumsum(new).tolist()
    ring = -(-(window + max(new) - 1) // PAGE) * PAGE
    for r in (ring, 0):
        table, n_pages = make_table(ends, r, rng)
        pages = make_pages(table, n_pages, ends, r, kv, dim, fmt, gen)
        q = (torch.randn(cu[-1], heads, dim, generator=gen) * 1.5).to(dtype).to(DEV)
        got = run_attention(q, pages, cu, ends, table, r, heads, kv, dim, window, dim ** -0.5)
        want, *sizes = plain.attention(q, pages, cu, ends, table, r, heads, kv, window, dim ** -0.5)
        tol = plain.attention_tolerance(want, *sizes, dtype, dim, fmt)
        assert ((got.double().cpu() - want).abs() <= tol).all()


@FORMATS
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
def test_scales_may_differ_by_many_powers_of_two(dtype, dim, fmt):
    """A sink whose value is nothing, values of any size beside it, and vectors of zeros."""
    heads, kv = 6, 2
    gen, rng = torch.Generator().manual_seed(23), np.random.RandomState(9)
    ends, cu = [300, 90], [0, 1, 4]
    table, n_pages = make_table(ends, 0, rng)
    pages = make_pages(table, n_pages, ends, 0, kv, dim, fmt, gen)
    stretch = torch.exp2(torch.rand(pages.v_scale.shape, generator=gen) * 60 - 30).to(DEV)
    pages = pages._replace(v_scale=pages.v_scale * stretch)
    first = table[0][0]
    zero, tiny = plain.quantise(torch.zeros(kv, dim), fmt)
    pages.v[first, :, 0] = zero.to(DEV)
    pages.v_scale[first, :, 0] = tiny.to(DEV)
    pages.v_scale[first, :, 1] = 0.0                          # somebody else's way to say zeros
    q = (torch.randn(cu[-1], heads, dim, generator=gen) * 1.5).to(dtype).to(DEV)
    pages.k[first, :, 0] = pages.k[first, :, 2]
    got = run_attention(q, pages, cu, ends, table, 0, heads, kv, dim, 0, dim ** -0.5)
    want, *sizes = plain.attention(q, pages, cu, ends, table, 0, heads, kv, 0, dim ** -0.5)
    tol = plain.attention_tolerance(want, *sizes, dtype, dim, fmt)
    assert ((got.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 96)])
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -20, 2.0 ** 60])
def test_queries_of_any_size(size, dtype, dim):
    """(Scores are brought back to order by the scale.)"""
    heads, kv, fmt = 4, 2, torch.int8
    gen, rng = torch.Generator().manual_seed(29), np.random.RandomState(9)
    ends, cu = [130], [0, 3]
    table, n_pages = make_table(ends, 0, rng)
    pages = make_pages(table, n_pages, ends, 0, kv, dim, fmt, gen)
    q = (torch.randn(cu[-1], heads, dim, generator=gen) * size).to(dtype).to(DEV)
    scale = dim ** -0.5 / size
    got = run_attention(q, pages, cu, ends, table, 0, heads, kv, dim, 0, scale)
    want, *sizes = plain.attention(q, pages, cu, ends, table, 0, heads, kv, 0, scale)
    tol = plain.attention_tolerance(want, *sizes, dtype, dim, fmt)
    assert ((got.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("count", [1, 4, 20])
def test_nan_stays_with_those_who_see_it(count, dtype, dim):
    heads, kv, fmt = 6, 2, torch.float8_e4m3fn
    gen, rng = torch.Generator().manual_seed(31), np.random.RandomState(2)
    ends, cu = [400 + count, 77 + count, 64], [0, count, 2 * count, 2 * count + 1]
    table, n_pages = make_table(ends, 0, rng)
    pages = make_pages(table, n_pages, ends, 0, kv, dim, fmt, gen)
    q = (torch.randn(cu[-1], heads, dim, generator=gen)).to(dtype).to(DEV)
    clean = run_attention(q, pages, cu, ends, table, 0, heads, kv, dim, 0, 0.1)
    # the second row's last token has a key of NaN in head 1 and a value of NaN in head 0
    pos = ends[1] - 1
    page = table[1][pos // PAGE]
    pages.k_scale[page, 1, pos % PAGE] = float("nan")
    pages.v_scale[page, 0, pos % PAGE] = float("nan")
    q[2 * count, 5, 3] = float("inf")                         # and the third row a query with an infinity
    got = run_attention(q, pages, cu, ends, table, 0, heads, kv, dim, 0, 0.1)
    sees = 2 * count - 1
    assert torch.isnan(got[sees]).all()
    assert torch.isnan(got[2 * count, 5]).all()
    same = torch.ones(got.shape[:2], dtype=torch.bool, device=DEV)
    same[sees] = False
    same[2 * count, 5] = False
    assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float32, 32)])
def test_rows_that_see_nothing_and_rows_of_no_tokens(dtype, dim):
    heads, kv, fmt = 4, 2, torch.int8
    gen, rng = torch.Generator().manual_seed(1), np.random.RandomState(2)
    ends, cu = [5, 0, 80, 1], [0, 2, 4, 4, 7]                 # rows 1 and 3 bring tokens before position 0
    table, n_pages = make_table(ends, 0, rng)
    pages = make_pages(table, n_pages, ends, 0, kv, dim, fmt, gen)
    q = torch.randn(9, heads, dim, generator=gen).to(dtype).to(DEV)
    out = torch.full_like(q, 7.0)
    st = status_word()
    K.attention_paged_q8(q, pages, ints(cu), ints(ends), ints(table), len(table[0]), 0, out, 3, 80, heads, kv, dim, 0,
                         0.2, st)
    want, *sizes = plain.attention(q, pages, cu, ends, table, 0, heads, kv, 0, 0.2)
    tol = plain.attention_tolerance(want, *sizes, dtype, dim, fmt)
    assert ((out.double().cpu() - want).abs() <= tol)[:7].all()
    assert (out[2:4] == 0).all() and (out[4:6] == 0).all()
    assert (out[7:] == 7.0).all()                             # behind the last row: as they were
    assert int(st.item()) == 0


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_tokens_of_other_rows_are_left_alone_where_keys_are_split(dtype, dim):
    """A call over some rows of a step: tokens in front of the first and behind the last stay as they are."""
    heads, kv, fmt = 4, 2, torch.int8
    gen, rng = torch.Generator().manual_seed(1), np.random.RandomState(2)
    ends, cu = [2000, 1500], [2, 3, 5]
    table, n_pages = make_table(ends, 0, rng)
    pages = make_pages(table, n_pages, ends, 0, kv, dim, fmt, gen)
    q = torch.randn(8, heads, dim, generator=gen).to(dtype).to(DEV)
    assert dtype == torch.bfloat16 or K.attention_q8_plan(8, 2, 2, 2000, heads, kv, dim, dtype)[0] > 0
    out = torch.full_like(q, 7.0)
    K.attention_paged_q8(q, pages, ints(cu), ints(ends), ints(table), len(table[0]), 0, out, 2, 2000, heads, kv, dim, 0,
                         0.2, status_word())
    assert (out[:2] == 7.0).all() and (out[5:] == 7.0).all()
    want, *sizes = plain.attention(q, pages, cu, ends, table, 0, heads, kv, 0, 0.2)
    tol = plain.attention_tolerance(want, *sizes, dtype, dim, fmt)
    assert ((out.double().cpu() - want).abs() <= tol)[2:5].all()


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_a_page_that_is_not_there_is_not_read(dtype, dim):
    heads, kv, fmt = 4, 2, torch.int8
    gen, rng = torch.Generator().manual_seed(1), np.random.RandomState(2)
    ends, cu = [200, 100], [0, 1, 2]
    table, n_pages = make_table(ends, 0, rng)
    pages = make_pages(table, n_pages, ends, 0, kv, dim, fmt, gen)
    q = torch.randn(2, heads, dim, generator=gen).to(dtype).to(DEV)
    clean = run_attention(q, pages, cu, ends, table, 0, heads, kv, dim, 0, 0.2)
    for bad in (-1, n_pages, 2 ** 31 - 1):
        broken = [list(r) for r in table]
        broken[0][1] = bad
        st = status_word()
        got = run_attention(q, pages, cu, ends, broken, 0, heads, kv, dim, 0, 0.2, status=st)
        assert int(st.item()) == 2
        assert torch.isfinite(got).all() and torch.equal(got[1], clean[1])
    # a length beyond the table (the row then sees the rest of its last page too, whatever that holds)
    # (the other row is compared bit for bit with a call of the same bound: that decides how keys are split)
    st, bound = status_word(), 200 + 64 * len(table[0])
    clean = run_attention(q, pages, cu, ends, table, 0, heads, kv, dim, 0, 0.2, max_end=bound)
    got = run_attention(q, pages, cu, [bound, 100], table, 0, heads, kv, dim, 0, 0.2, status=st)
    assert int(st.item()) == 2 and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("longest", [200, 4000, 40000])
@pytest.mark.parametrize("window", [0, 70])
def test_lengths_and_offsets_that_are_anything(longest, window, dtype, dim):
    """What the device gives as lengths and offsets is brought inside the page table and the tokens."""
    heads, kv, fmt, big = 4, 2, torch.int8, 2 ** 31 - 1
    gen, rng = torch.Generator().manual_seed(1), np.random.RandomState(2)
    ends = [longest, 90, 80, 150, 33, 20]
    table, n_pages = make_table(ends, 0, rng)
    pages = make_pages(table, n_pages, ends, 0, kv, dim, fmt, gen)
    q = torch.randn(6, heads, dim, generator=gen).to(dtype).to(DEV)
    cu = [0, 1, 2, 3, 4, 5, 6]
    want, *sizes = plain.attention(q, pages, cu, ends, table, 0, heads, kv, window, 0.2)
    tol = plain.attention_tolerance(want, *sizes, dtype, dim, fmt)

    def call(cu, ends):
        out, st = torch.full_like(q, 7.0), status_word()
        K.attention_paged_q8(q, pages, ints(cu), ints(ends), ints(table), len(table[0]), 0, out, 1, longest, heads, kv,
                             dim, window, 0.2, st)
        return out, (out.double().cpu() - want).abs() <= tol, int(st.item())
    for wild in (big, big - 31, 2 ** 30, 64 * len(table[0]) + 1):
        out, right, st = call(cu, [ends[0], wild, ends[2], wild, ends[4], ends[5]])
        assert st == 2 and right[[0, 2, 4, 5]].all()
    for wild in (-1, -2 ** 31, -2 ** 31 + 40):
        out, right, st = call(cu, [ends[0], wild, ends[2], wild, ends[4], ends[5]])
        assert st == 0 and right[[0, 2, 4, 5]].all() and (out[[1, 3]] == 0).all()
    for wild in (-1, -2 ** 31, 7, big):
        out, right, st = call([0, 1, wild, 3, 4, 5, 6], ends)
        assert st == 0 and right[[0, 3, 4, 5]].all() and (out[1:3] == 7.0).all()


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_offsets_beyond_32_bits(dtype, dim):
    heads, kv, fmt = 8, 8, torch.int8
    n_pages = 2 ** 32 // (kv * PAGE * dim) + 3
    codes = [torch.zeros((n_pages, kv, PAGE, dim), dtype=torch.int8, device=DEV) for _ in range(2)]
    scales = [torch.zeros((n_pages, kv, PAGE), dtype=torch.float32, device=DEV) for _ in range(2)]
    pages = K.Q8Pages(codes[0], codes[1], scales[0], scales[1])
    table = [[n_pages - 1, n_pages - 2]]
    gen = torch.Generator().manual_seed(3)
    small = []
    for i in range(2):
        c, s = plain.quantise(torch.randn(2, kv, PAGE, dim, generator=gen), fmt)
        codes[i][n_pages - 2:] = c.to(DEV)
        scales[i][n_pages - 2:] = s.to(DEV)
        small.append((c, s))
    q = torch.randn(1, heads, dim, generator=gen).to(dtype).to(DEV)
    got = run_attention(q, pages, [0, 1], [100], table, 0, heads, kv, dim, 0, dim ** -0.5)
    tiny = K.Q8Pages(small[0][0], small[1][0], small[0][1], small[1][1])
    want, *sizes = plain.attention(q, tiny, [0, 1], [100], [[1, 0]], 0, heads, kv, 0, dim ** -0.5)
    assert ((got.double().cpu() - want).abs() <= plain.attention_tolerance(want, *sizes, dtype, dim, fmt)).all()
    out = [torch.empty((2, kv, PAGE, dim), dtype=dtype, device=DEV) for _ in range(2)]
    K.read_pages_q8(pages, ints(table), 2, 0, ints([100]), out[0], out[1], status_word())
    assert torch.equal(out[1][0].cpu(), (small[1][0][1].float() * small[1][1][1].unsqueeze(-1)).to(dtype))


@FORMATS
@pytest.mark.parametrize("dtype,dim", [(torch.float32, 16), (torch.float32, 64), (torch.float32, 112), (torch.float32, 128),
                                       (torch.float32, 192), (torch.float32, 256), (torch.bfloat16, 96)])
@pytest.mark.parametrize("rows,heads,kv,window", [
    ([(4, 300), (3, 261), (1, 310), (0, 5), (4, 0), (4, 60), (2, 255), (4, 256)], 40, 8, 0), ([(10, 4990), (7, 13)], 4, 2, 0),
    ([(40, 290)] * 4, 12, 12, 130), ([(4, 600)] * 16, 20, 4, 200)], ids=str)
def test_attention_of_many_rows_on_the_fp32_pipe(rows, heads, kv, window, dtype, dim, fmt):
    new, past = zip(*rows)
    ends, cu = [n + p for n, p in zip(new, past)], [0] + np.cumsum(new).tolist()
    ring = -(-(window + max(new) - 1) // PAGE) * PAGE if window else 0
    gen, rng = torch.Generator().manual_seed(dim), np.random.RandomState(6)
    table, n_pages = make_table(ends, ring, rng)
    pages = make_pages(table, n_pages, ends, ring, kv, dim, fmt, gen)
    q = torch.randn(cu[-1], heads, dim, generator=gen).to(dtype).to(DEV)
    # what decides that a block takes 32 rows
    span = max(ends) if not window else min(max(ends), window + max(new) + PAGE - 1)
    blocks = len(rows) * kv * -(-max(new) * (heads // kv) // 32)
    assert max(new) * (heads // kv) > 12 and blocks * -(-span // PAGE) >= 2 * K.sm_count(q.device)
    got = run_attention(q, pages, cu, ends, table, ring, heads, kv, dim, window, dim ** -0.5)
    want, *sizes = plain.attention(q, pages, cu, ends, table, ring, heads, kv, window, dim ** -0.5)
    tol = plain.attention_tolerance(want, *sizes, dtype, dim, fmt)
    assert ((got.double().cpu() - want).abs() <= tol).all()
    # a value of NaN at the first row's last position but one: the last two tokens of its head group see it
    place = (ends[0] - 2) % ring if ring else ends[0] - 2
    pages.v_scale[table[0][place // PAGE], 0, place % PAGE] = float("nan")
    again = run_attention(q, pages, cu, ends, table, ring, heads, kv, dim, window, dim ** -0.5)
    hit = torch.zeros(cu[-1], heads, dtype=torch.bool, device=DEV)
    hit[new[0] - 2:new[0], :heads // kv] = True
    assert torch.isnan(again[hit]).all() and torch.equal(again[~hit], got[~hit])


@FORMATS
@pytest.mark.parametrize("heads,kv,dim", [(6, 2, 128), (5, 1, 64)])
@pytest.mark.parametrize("rows,window,spread", [
    ([(300, 1000)], 0, 0.0), ([(1, 5), (257, 0), (128, 4000), (129, 127), (2, 0)], 0, 8.0), ([(64, 64)] * 5, 0, 0.0),
    ([(400, 900), (1, 300), (100, 28)], 130, 8.0), ([(513, 511)], 1, 0.0)], ids=str)
def test_portions_on_tcgen05(rows, window, spread, heads, kv, dim, fmt, monkeypatch):
    """Keys, values and probabilities are halves there: eight times as exact as bfloat16."""
    monkeypatch.setattr(K, "q8_on_tcgen05", lambda *a: True)
    gen, rng = torch.Generator().manual_seed(43), np.random.RandomState(6)
    new, past = zip(*rows)
    ends, cu = [n + p for n, p in zip(new, past)], [0] + np.cumsum(new).tolist()
    ring = -(-(window + max(new) - 1) // PAGE) * PAGE if window else 0
    table, n_pages = make_table(ends, ring, rng)
    pages = make_pages(table, n_pages, ends, ring, kv, dim, fmt, gen, spread)
    q = torch.randn(cu[-1], heads, dim, generator=gen).to(torch.bfloat16).to(DEV)
    most = float(pages.v_scale.nan_to_num(0.0).max()) * plain.LIMIT[fmt]
    for scale in (dim ** -0.5, -0.02, 0.0):
        got = run_attention(q, pages, cu, ends, table, ring, heads, kv, dim, window, scale)
        want, *sizes = plain.attention(q, pages, cu, ends, table, ring, heads, kv, window, scale)
        tol = plain.halves_tolerance(want, *sizes, most)
        assert ((got.double().cpu() - want).abs() <= tol).all()
        again = run_attention(q, pages, cu, ends, table, ring, heads, kv, dim, window, scale)
        assert torch.equal(got, again)


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 16), (torch.bfloat16, 64)])
def test_more_blocks_than_a_grid_has_rows(dtype, dim, monkeypatch):
    """A long portion of very many heads: items beyond 65,535."""
    monkeypatch.setattr(K, "q8_on_tcgen05", lambda *a: False)
    heads, n, fmt = 1040, 2050, torch.int8
    gen, rng = torch.Generator().manual_seed(1), np.random.RandomState(2)
    table, n_pages = make_table([n], 0, rng)
    pages = make_pages(table, n_pages, [n], 0, heads, dim, fmt, gen, junk=False)
    q = torch.randn(n, heads, dim, generator=gen).to(dtype).to(DEV)
    got = run_attention(q, pages, [0, n], [n], table, 0, heads, heads, dim, 0, 0.2)
    order = ints(table[0]).long()
    sees = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
    for h in (0, 517, 1039):
        k, v = ((c[order, h].double() * s[order, h].double().unsqueeze(-1)).reshape(-1, dim)[:n]
                for c, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)))
        s = (q[:, h].double() @ k.T * 0.2).masked_fill(~sees, -np.inf)
        p = torch.softmax(s, -1)
        size = (q[:, h].double().abs() @ k.abs().T * 0.2).masked_fill(~sees, 0.0).amax(-1)
        top = (p * pages.v_scale[order, h].double().reshape(-1)[:n]).amax(-1)
        keys = torch.arange(1, n + 1, device=DEV).double()
        want, mass = p @ v, p @ v.abs()
        tol = plain.attention_tolerance(want.unsqueeze(1), mass.unsqueeze(1), top.unsqueeze(1), size.unsqueeze(1), keys,
                                        dtype, dim, fmt)
        assert ((got[:, h].double() - want).abs() <= tol[:, 0]).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [0, 70, 500])
def test_lengths_and_offsets_that_are_anything_on_tcgen05(window, dim, monkeypatch):
    monkeypatch.setattr(K, "q8_on_tcgen05", lambda *a: True)
    heads, kv, fmt, big, longest = 4, 2, torch.int8, 2 ** 31 - 1, 4000
    gen, rng = torch.Generator().manual_seed(1), np.random.RandomState(2)
    ends, new = [longest, 90, 180, 650, 33, 320], [40, 3, 130, 40, 1, 300]
    cu = [0] + np.cumsum(new).tolist()
    table, n_pages = make_table(ends, 0, rng)
    pages = make_pages(table, n_pages, ends, 0, kv, dim, fmt, gen)
    q = torch.randn(cu[-1], heads, dim, generator=gen).to(torch.bfloat16).to(DEV)
    want, *sizes = plain.attention(q, pages, cu, ends, table, 0, heads, kv, window, 0.2)
    most = float(pages.v_scale.nan_to_num(0.0).max()) * plain.LIMIT[fmt]
    tol = plain.halves_tolerance(want, *sizes, most)

    def call(cu, ends, most_new=300):
        out, st = torch.full_like(q, 7.0), status_word()
        K.attention_paged_q8(q, pages, ints(cu), ints(ends), ints(table), len(table[0]), 0, out, most_new, longest, heads,
                             kv, dim, window, 0.2, st)
        return out, (out.double().cpu() - want).abs() <= tol, int(st.item())

    def rows(x, which):
        return torch.cat([x[cu[b]:cu[b + 1]] for b in which])
    out, right, st = call(cu, ends)
    assert st == 0 and right.all()
    for wild in (big, big - 31, 2 ** 30, longest + 1):
        out, right, st = call(cu, [ends[0], wild, ends[2], wild, ends[4], ends[5]])
        assert st == 2 and rows(right, [0, 2, 4, 5]).all()
    for wild in (-1, -2 ** 31, -2 ** 31 + 40):
        out, right, st = call(cu, [ends[0], wild, ends[2], wild, ends[4], ends[5]])
        assert st == 0 and rows(right, [0, 2, 4, 5]).all() and (rows(out, [1, 3]) == 0).all()
    for wild in (-1, -2 ** 31, cu[-1] + 1, big):
        broken = list(cu)
        broken[2] = wild
        out, right, st = call(broken, ends)
        assert st == 0 and rows(right, [0, 3, 4, 5]).all() and (rows(out, [1, 2]) == 7.0).all()
    # a row that brings more tokens than was said, and pages that are not there
    out, right, st = call(cu, ends, most_new=64)
    assert rows(right, [0, 1, 3, 4]).all()
    for bad in (-1, n_pages, big):
        broken = [list(r) for r in table]
        broken[0][-1] = broken[2][0] = bad
        out, st = torch.full_like(q, 7.0), status_word()
        K.attention_paged_q8(q, pages, ints(cu), ints(ends), ints(broken), len(table[0]), 0, out, 300, longest, heads, kv,
                             dim, window, 0.2, st)
        assert int(st.item()) == 2
        assert rows((out.double().cpu() - want).abs() <= tol, [1, 3, 4, 5]).all() and torch.isfinite(out).all()


@FORMATS
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("high", [10, 40, 80])
@pytest.mark.parametrize("what", ["keys", "values", "both"])
def test_a_later_token_far_above_the_others(what, high, dim, fmt, monkeypatch):
    """Tokens in front of one whose key or value is 2^high times as large do not notice; the others see it."""
    monkeypatch.setattr(K, "q8_on_tcgen05", lambda *a: True)
    heads, kv = 4, 2
    gen, rng = torch.Generator().manual_seed(1), np.random.RandomState(2)
    ends, cu, at = [700], [0, 300], 560                       # position 560 is the token 160
    table, n_pages = make_table(ends, 0, rng)
    pages = make_pages(table, n_pages, ends, 0, kv, dim, fmt, gen)
    q = torch.randn(cu[-1], heads, dim, generator=gen).to(torch.bfloat16).to(DEV)
    page, place = table[0][at // PAGE], at % PAGE
    if what != "values":
        pages.k_scale[page, :, place] *= 2.0 ** high
    if what != "keys":
        pages.v_scale[page, :, place] *= 2.0 ** high
    got = run_attention(q, pages, cu, ends, table, 0, heads, kv, dim, 0, 0.1)
    want, *sizes = plain.attention(q, pages, cu, ends, table, 0, heads, kv, 0, 0.1)
    # (where the far value is seen its weight is most of the result)
    most = torch.zeros(cu[-1], 1, dtype=torch.float64)
    ordinary = pages.v_scale.nan_to_num(0.0).clone()
    ordinary[page, :, place] = 0
    most[:160] = float(ordinary.max()) * plain.LIMIT[fmt]
    most[160:] = float(pages.v_scale.nan_to_num(0.0).max()) * plain.LIMIT[fmt]
    tol = plain.halves_tolerance(want, *sizes, most)
    assert ((got.double().cpu() - want).abs() <= tol).all()


@FORMATS
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 96)])
@pytest.mark.parametrize("high", [10, 40, 80])
@pytest.mark.parametrize("longest", [300, 40000])
def test_a_later_draft_with_a_key_far_above_the_others(longest, high, dtype, dim, fmt):
    heads, kv = 4, 2
    gen, rng = torch.Generator().manual_seed(1), np.random.RandomState(2)
    ends, cu, at = [300, 100], [0, 6, 12], 297                # position 297 is the row's fourth token
    table, n_pages = make_table(ends, 0, rng)
    pages = make_pages(table, n_pages, ends, 0, kv, dim, fmt, gen)
    q = torch.randn(cu[-1], heads, dim, generator=gen).to(dtype).to(DEV)
    pages.k_scale[table[0][at // PAGE], :, at % PAGE] *= 2.0 ** high
    got = run_attention(q, pages, cu, ends, table, 0, heads, kv, dim, 0, 0.1, max_end=longest)
    want, *sizes = plain.attention(q, pages, cu, ends, table, 0, heads, kv, 0, 0.1)
    tol = plain.attention_tolerance(want, *sizes, dtype, dim, fmt)
    assert ((got.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("heads", [6, 40])
def test_portions_captured_twice_and_on_another_stream(heads, monkeypatch):
    monkeypatch.setattr(K, "q8_on_tcgen05", lambda *a: True)
    kv, dim, fmt = 2, 128, torch.float8_e4m3fn
    gen, rng = torch.Generator().manual_seed(1), np.random.RandomState(2)
    ends, cu = [1500, 900, 64], [0, 300, 333, 397]
    table, n_pages = make_table(ends, 0, rng)
    pages = make_pages(table, n_pages, ends, 0, kv, dim, fmt, gen)
    qs = [torch.randn(cu[-1], heads, dim, generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2)]
    eager = [run_attention(q, pages, cu, ends, table, 0, heads, kv, dim, 0, 0.1) for q in qs]
    cu_d, end_d, table_d, st = ints(cu), ints(ends), ints(table), status_word()
    torch.cuda.synchronize()

    def call(q, out):
        K.attention_paged_q8(q, pages, cu_d, end_d, table_d, len(table[0]), 0, out, 300, 1500, heads, kv, dim, 0, 0.1, st)
    outs, graphs = [], []
    for q in qs:
        out, graph = torch.zeros_like(q), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            call(q, out)
        outs.append(out)
        graphs.append(graph)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, eager))
    # two calls at once
    sides, outs = [torch.cuda.Stream() for _ in qs], [torch.zeros_like(q) for q in qs]
    for side, q, out in zip(sides, qs, outs):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                call(q, out)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, eager)) and int(st.item()) == 0


@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("back", [True, False])
def test_a_page_table_wider_than_its_rows(window, back, monkeypatch):
    """Places that no position of a row can lie in cost nothing and change nothing; a length beyond ``max_end``
    is reported where that sizes what is read back."""
    monkeypatch.setattr(K, "q8_on_tcgen05", lambda *a: back)
    heads, kv, dim, fmt = 6, 2, 128, torch.int8
    gen, rng = torch.Generator().manual_seed(41), np.random.RandomState(6)
    ends, cu = [140, 75, 33], [0, 40, 108, 141]
    ring = 192 if window else 0
    table, n_pages = make_table(ends, ring, rng)
    pages = make_pages(table, n_pages, ends, ring, kv, dim, fmt, gen)
    q = torch.randn(cu[-1], heads, dim, generator=gen).to(torch.bfloat16).to(DEV)
    clean = run_attention(q, pages, cu, ends, table, ring, heads, kv, dim, window, 0.1)
    wide = [r + [n_pages + 7] * 4000 for r in table]
    before = torch.cuda.max_memory_allocated()
    assert torch.equal(run_attention(q, pages, cu, ends, wide, ring, heads, kv, dim, window, 0.1), clean)
    assert torch.cuda.max_memory_allocated() - before < 2 ** 24
    if back and not window:
        st = status_word()
        run_attention(q, pages, cu, ends, table, ring, heads, kv, dim, window, 0.1, status=st, max_end=100)
        assert int(st.item()) & 2


def test_captured_twice_and_on_another_stream():
    heads, kv, dim, fmt = 28, 4, 128, torch.float8_e4m3fn
    gen, rng = torch.Generator().manual_seed(1), np.random.RandomState(2)
    ends, cu = [1500, 900], [0, 1, 2]
    table, n_pages = make_table(ends, 0, rng)
    pages = make_pages(table, n_pages, ends, 0, kv, dim, fmt, gen)
    qs = [torch.randn(2, heads, dim, generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2)]
    eager = [run_attention(q, pages, cu, ends, table, 0, heads, kv, dim, 0, 0.1) for q in qs]
    cu_d, end_d, table_d, st = ints(cu), ints(ends), ints(table), status_word()
    torch.cuda.synchronize()
    outs, graphs = [], []
    for q in qs:
        out, graph = torch.zeros_like(q), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            K.attention_paged_q8(q, pages, cu_d, end_d, table_d, len(table[0]), 0, out, 1, 1500, heads, kv, dim, 0, 0.1, st)
        outs.append(out)
        graphs.append(graph)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, eager))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = torch.zeros_like(qs[0])
        K.attention_paged_q8(qs[0], pages, cu_d, end_d, table_d, len(table[0]), 0, out, 1, 1500, heads, kv, dim, 0, 0.1, st)
    side.synchronize()
    assert torch.equal(out, eager[0])


@FORMATS
@pytest.mark.parametrize("heads,kv,dim", [(6, 2, 128), (14, 2, 64), (3, 3, 64)])
@pytest.mark.parametrize("rows,window", [([(40, 0)], 0), ([(100, 29), (1, 300), (33, 64), (129, 0)], 0),
                                         ([(70, 500), (64, 0), (3, 127)], 90)])
@pytest.mark.parametrize("at_a_time", [None, 2])
def test_portions_some_rows_at_a_time(rows, window, heads, kv, dim, fmt, at_a_time, monkeypatch):
    """The other way to attend, which long portions take: the same result, NaN with those who see it only
    (a value of NaN in a later token, in another row, in a place no row sees), in one go and some rows at a
    time."""
    monkeypatch.setattr(K, "q8_on_tcgen05", lambda *a: True)
    gen, rng = torch.Generator().manual_seed(41), np.random.RandomState(6)
    new, past = zip(*rows)
    ends = [n + p for n, p in zip(new, past)]
    cu = [0] + np.cumsum(new).tolist()
    ring = -(-(window + max(new) - 1) // PAGE) * PAGE if window else 0
    table, n_pages = make_table(ends, ring, rng)
    if at_a_time:
        monkeypatch.setattr(K, "Q8_PORTION_BYTES", at_a_time * (len(table[0]) + 1) * kv * PAGE * dim * 4)
    pages = make_pages(table, n_pages, ends, ring, kv, dim, fmt, gen)
    q = torch.randn(cu[-1], heads, dim, generator=gen).to(torch.bfloat16).to(DEV)
    most = float(pages.v_scale.nan_to_num(0.0).max()) * plain.LIMIT[fmt]
    got = run_attention(q, pages, cu, ends, table, ring, heads, kv, dim, window, dim ** -0.5)
    want, *sizes = plain.attention(q, pages, cu, ends, table, ring, heads, kv, window, dim ** -0.5)
    tol = plain.halves_tolerance(want, *sizes, most)
    assert ((got.double().cpu() - want).abs() <= tol).all()
    # a value of NaN at the first row's last position but one: its last two tokens see it
    pos = ends[0] - 2
    place = pos % ring if ring else pos
    page = table[0][place // PAGE]
    pages.v_scale[page, 0, place % PAGE] = float("nan")
    pages.k_scale[page, kv - 1, place % PAGE] = float("nan")
    bad = run_attention(q, pages, cu, ends, table, ring, heads, kv, dim, window, dim ** -0.5)
    group = heads // kv
    sees = torch.zeros(got.shape[:2], dtype=torch.bool)
    sees[new[0] - 2:new[0], :group] = True
    sees[new[0] - 2:new[0], (kv - 1) * group:] = True
    assert torch.isnan(bad[sees.to(DEV)]).all()
    assert torch.equal(bad[~sees.to(DEV)], got[~sees.to(DEV)])


# ---- written and read back ------------------------------------------------------------------------
def rotated(x, positions, inv_freq, rotary, style, heads_qk):
    """float64 q and k of ``x`` [tokens, all heads, dim], the first ``heads_qk`` rotated."""
    y = x.clone()
    if inv_freq is None:
        return y
    angle = positions.double().unsqueeze(1) * inv_freq
    cos, sin = angle.cos().unsqueeze(1), angle.sin().unsqueeze(1)
    h = rotary // 2
    a = slice(0, h) if style == 0 else slice(0, rotary, 2)
    b = slice(h, rotary) if style == 0 else slice(1, rotary, 2)
    lo, hi = x[:, :heads_qk, a], x[:, :heads_qk, b]
    y[:, :heads_qk, a], y[:, :heads_qk, b] = lo * cos - hi * sin, lo * sin + hi * cos
    return y


@FORMATS
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape,rotary,style", [((28, 4, 128), 128, 0), ((14, 2, 64), 64, 0), ((3, 1, 256), 256, 0),
                                                ((4, 2, 128), 64, 0), ((4, 2, 64), 64, 1), ((6, 3, 96), 48, 1),
                                                ((2, 1, 16), 0, 0)])
@pytest.mark.parametrize("rows,window", [([(1, 0)], 0), ([(1, 63), (1, 64), (3, 200)], 0), ([(150, 0), (70, 61)], 0),
                                         ([(1, 70), (90, 30)], 20)])
@pytest.mark.parametrize("splits", [0, 3])
def test_written_and_read_back(shape, rotary, style, rows, window, splits, dtype, fmt):
    heads, kv, dim = shape
    gen, rng = torch.Generator().manual_seed(17), np.random.RandomState(4)
    new, past = zip(*rows)
    ends = [n + p for n, p in zip(new, past)]
    n = sum(new)
    ring = -(-(window + 1) // PAGE) * PAGE if window else 0   # shorter than the longest row: part of it is not kept
    table, n_pages = make_table(ends, ring, rng)
    pages = make_pages(table, n_pages, ends, ring, kv, dim, fmt, gen, junk=False)
    before = [t.clone() for t in pages]
    width = (heads + 2 * kv) * dim
    x = torch.randn((splits, n, width) if splits else (n, width), generator=gen)
    x[..., width // 2] *= 40.0                                # an outlier channel
    bias = torch.randn(width, generator=gen) if splits else None
    positions = [p + i for c, p in rows for i in range(c)]
    token_row = [b for b, c in enumerate(new) for _ in range(c)]
    inv = (1e4 ** (-2.0 * torch.arange(rotary // 2, dtype=torch.float64) / max(1, rotary))) if rotary else None
    q = torch.empty((n, heads, dim), dtype=dtype, device=DEV)
    k, v = (torch.empty((n, kv, dim), dtype=dtype, device=DEV) for _ in range(2))
    st = status_word()
    K.rope_kvstore_q8(x.to(DEV), ints(positions), ints(token_row), ints(ends), None if inv is None else inv.to(DEV),
                      q, k, v, pages, ints(table), len(table[0]), ring, heads, kv, dim, rotary, style, st,
                      n_partials=splits, bias=None if bias is None else bias.to(DEV))
    back = [torch.empty((len(rows) * len(table[0]), kv, PAGE, dim), dtype=torch.float32, device=DEV) for _ in range(2)]
    K.read_pages_q8(pages, ints(table), len(table[0]), ring, ints(ends), back[0], back[1], st)
    assert int(st.item()) == 0
    x64 = x.double()
    x64 = (x64.sum(0) if splits else x64) + (bias.double() if bias is not None else 0)
    x64 = x64.view(n, heads + 2 * kv, dim)
    y = rotated(x64, torch.tensor(positions), inv, rotary, style, heads + kv)
    # float32 sums of up to splits + 1 terms, then two products and a sum, with a sine and cosine of
    # a float32 angle in [0, 2 pi): a few 2^-24 of the pair's size, 8 of them are allowed here
    pair = torch.maximum(x64.abs(), y.abs()).amax(-1, keepdim=True).expand_as(y) * (splits + 8) * 2.0 ** -24 * 4
    rounding = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    for got, want, off in ((q, y[:, :heads], pair[:, :heads]), (k, y[:, heads:heads + kv], pair[:, heads:heads + kv]),
                           (v, y[:, heads + kv:], pair[:, heads + kv:])):
        assert ((got.double().cpu() - want).abs() <= want.abs() * rounding + off).all()
    written = torch.zeros(n_pages, PAGE, dtype=torch.bool)
    for which, src, off in ((0, y[:, heads:heads + kv], pair[:, heads:heads + kv]), (1, y[:, heads + kv:], pair[:, heads + kv:])):
        codes, scales = pages[which].cpu(), pages[2 + which].cpu()
        for t in range(n):
            b, p = token_row[t], positions[t]
            if ring and p < ends[b] - ring:
                continue
            place = p % ring if ring else p
            page = table[b][place // PAGE]
            written[page, place % PAGE] = True
            a = src[t].abs().amax(-1)
            s = scales[page, :, place % PAGE].double()
            assert ((s * plain.LIMIT[fmt] - a).abs() <= a * 2.0 ** -22 + off[t].amax(-1)).all()
            held = plain.values(codes[page, :, place % PAGE], scales[page, :, place % PAGE])
            limit = plain.half_step(src[t], s, fmt) * (1 + 2.0 ** -12) + off[t] + src[t].abs() * 2.0 ** -22
            assert ((held - src[t]).abs() <= limit).all()
            # read back: code times scale, rounded once
            at = b * len(table[0]) + place // PAGE
            assert torch.equal(back[which][at, :, place % PAGE].cpu(),
                               codes[page, :, place % PAGE].float() * scales[page, :, place % PAGE].unsqueeze(-1))
    # nothing else of the pages has changed
    keep = ~written.unsqueeze(1).expand(n_pages, kv, PAGE)
    for which in range(2):
        assert torch.equal(pages[which].cpu().view(torch.uint8)[keep], before[which].cpu().view(torch.uint8)[keep])
        assert torch.equal(pages[2 + which].cpu()[keep], before[2 + which].cpu()[keep])


@FORMATS
def test_codes_are_the_definitions(fmt):
    """Values (not rotated, not summed) have exactly the codes and scales that the definition gives in
    float32: at every power of two, of zeros, of the smallest and largest numbers."""
    kv, dim, n = 1, 128, 64
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(n, dim, generator=gen) * torch.exp2(torch.arange(n) * 4.0 - 126.0).unsqueeze(1)
    x[0] = 0.0
    x[1, 1:] = 0.0
    x[2] = -x[2].abs()
    x[3] = torch.arange(dim) * 2.0 ** -149                    # below the normal range
    x[4, 5], x[5, 7] = float("inf"), float("nan")
    x[6, :64] = x[6, 64:] * 2.0 ** -9                          # subnormal codes
    qkv = torch.cat([torch.zeros(n, 2 * dim), x], 1).to(DEV)
    pages = K.q8_pages(1, kv, dim, fmt)
    q, k, v = (torch.empty((n, 1, dim), device=DEV) for _ in range(3))
    st = status_word()
    K.rope_kvstore_q8(qkv, ints(list(range(n))), ints([0] * n), ints([n]), None, q, k, v, pages, ints([0]), 1, 0, 1, 1,
                      dim, 0, 0, st)
    code, scale = plain.quantise(x, fmt)
    assert torch.equal(pages.v_scale[0, 0, :n].cpu().view(torch.int32)[~torch.isnan(scale)],
                       scale.view(torch.int32)[~torch.isnan(scale)])
    assert torch.equal(torch.isnan(pages.v_scale[0, 0, :n].cpu()), torch.isnan(scale))
    assert torch.equal(pages.v[0, 0, :n].cpu().float(), code.float())
    assert torch.equal(v[:, 0].cpu().view(torch.int32)[~torch.isnan(x)], x.view(torch.int32)[~torch.isnan(x)])
    out = [torch.empty((1, 1, PAGE, dim), device=DEV) for _ in range(2)]
    K.read_pages_q8(pages, ints([0]), 1, 0, ints([n]), out[0], out[1], st)
    back = out[1][0, 0].cpu()
    assert torch.isnan(back[4:6]).all() and torch.isfinite(back[:4]).all()
    assert int(st.item()) == 0


@FORMATS
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("kv,dim", [(4, 128), (2, 64), (1, 16), (3, 96), (1, 256)])
@pytest.mark.parametrize("ring", [0, 128])
def test_read_back(kv, dim, ring, dtype, fmt):
    gen, rng = torch.Generator().manual_seed(13), np.random.RandomState(8)
    ends = [1, 64, 65, 200, 0, 127]
    table, n_pages = make_table(ends, ring, rng)
    pages = make_pages(table, n_pages, ends, ring, kv, dim, fmt, gen)
    wide = len(table[0])
    for fill in (True, False):
        out = [torch.full((len(ends) * wide, kv, PAGE, dim), 5.0, dtype=dtype, device=DEV) for _ in range(2)]
        st = status_word()
        K.read_pages_q8(pages, ints(table), wide, ring, ints(ends), out[0], out[1], st, fill=fill)
        assert int(st.item()) == 0
        for which in range(2):
            codes, scales = pages[which].cpu(), pages[2 + which].cpu()
            want = torch.zeros((len(ends) * wide, kv, PAGE, dim), dtype=dtype)
            for b, end in enumerate(ends):
                span = min(end, ring) if ring else end
                for i in range(wide):
                    n = min(PAGE, span - i * PAGE)
                    if n > 0:
                        page = table[b][i]
                        want[b * wide + i, :, :n] = (codes[page, :, :n].float() * scales[page, :, :n].unsqueeze(-1)).to(dtype)
                    elif not fill:
                        want[b * wide + i] = 5.0
            assert torch.equal(out[which].cpu(), want)
    broken = [list(r) for r in table]
    broken[3][1], broken[0][0] = n_pages, -7                  # pages that are needed and are none
    st = status_word()
    K.read_pages_q8(pages, ints(broken), wide, ring, ints(ends), out[0], out[1], st)
    assert int(st.item()) == 2
    assert (out[0][3 * wide + 1] == 0).all() and (out[0][0] == 0).all()
    assert torch.equal(out[0][2 * wide].cpu(), want[2 * wide]) or which == 1


def test_a_position_without_a_page_is_not_written():
    heads, kv, dim, fmt = 2, 1, 64, torch.int8
    pages = K.q8_pages(2, kv, dim, fmt)
    qkv = torch.randn(5, (heads + 2 * kv) * dim, device=DEV)
    q = torch.empty((5, heads, dim), device=DEV)
    st = status_word()
    # row 0 has page 1 for positions 0..63 and a page out of range behind it; row 1 has none
    table = [[1, 2], [-1, -1]]
    K.rope_kvstore_q8(qkv, ints([3, 64, 0, 128, -1]), ints([0, 0, 1, 0, 0]), ints([129, 1]), None, q, None, None, pages,
                      ints(table), 2, 0, heads, kv, dim, 0, 0, st)
    assert int(st.item()) == 2
    changed = (pages.v_scale != 0).nonzero().cpu().tolist()
    assert changed == [[1, 0, 3]]
    assert torch.equal(q.view(5, -1), qkv[:, :heads * dim])
