"""The 8-bit cache's bookkeeping, and sequences taken back (no GPU needed)."""
import pytest
import torch

from minfer_b200.cache.paged import PAGE, Cache, CacheError, GroupKey, cache_dtype_of


def make(dtype=torch.int8, max_tokens=1024, max_seqs=4, step_tokens=1):
    return Cache({0: GroupKey(2, 16, 0), 1: GroupKey(2, 16, 70), 2: GroupKey(2, 16, 70)}, max_tokens, max_seqs, dtype,
                 "cpu", step_tokens)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_scales_beside_the_codes(dtype):
    c = make(dtype)
    for g in c.groups:
        n = len(g.entries)
        assert g.k.dtype == g.v.dtype == dtype and g.k.shape == (n, g.n_pages + 1, 2, PAGE, 16)
        assert g.k_scale.shape == g.v_scale.shape == (n, g.n_pages + 1, 2, PAGE) and g.k_scale.dtype == torch.float32
        assert len({g.k.data_ptr(), g.v.data_ptr(), g.k_scale.data_ptr(), g.v_scale.data_ptr()}) == 4
        for t in (g.k, g.k_scale):                            # what the kernels ask of addresses
            assert all(t[i].data_ptr() % 16 == 0 for i in range(n))
    ks, vs = c.group_of[2].entry_scales(2)
    assert ks.data_ptr() == c.group_of[2].k_scale[1].data_ptr() and vs.shape == ks.shape
    assert c.bytes() == sum(len(g.entries) * g.n_pages * 2 * PAGE * 2 * (16 + 4) for g in c.groups)
    c.check_canaries()
    g = c.groups[1]
    g._guarded[3].raw[-1] = 0
    with pytest.raises(CacheError, match="scales of the values"):
        c.check_canaries()


def test_a_plain_cache_has_no_scales():
    c = make(torch.bfloat16)
    assert c.groups[0].entry_scales(0) == (None, None)
    assert c.bytes() == sum(len(g.entries) * g.n_pages * 2 * PAGE * 2 * 16 * 2 for g in c.groups)


@pytest.mark.parametrize("key", [GroupKey(2, 16, 0, 32), GroupKey(2, 16, 0, 16, True)])
def test_values_of_another_shape_are_refused(key):
    with pytest.raises(CacheError, match="8 bits"):
        Cache({0: key}, 64, 1, torch.int8, "cpu")


def test_names_of_the_types():
    from minfer_b200.cli import CliError, parse_args      # (here: what is imported first keeps its stdout)
    assert cache_dtype_of(None) is None
    assert cache_dtype_of("e4m3") is torch.float8_e4m3fn is cache_dtype_of(torch.float8_e4m3fn)
    assert cache_dtype_of("int8") is torch.int8
    for bad in ("bfloat16", torch.bfloat16, 8):
        with pytest.raises(CacheError, match="e4m3 or int8"):
            cache_dtype_of(bad)
    assert parse_args(["m", "1"])["cache_dtype"] is None
    assert parse_args(["m", "1", "--cache-dtype", "auto"])["cache_dtype"] is None
    assert parse_args(["m", "1", "--cache-dtype", "e4m3"])["cache_dtype"] == "e4m3"
    with pytest.raises(CliError):
        parse_args(["m", "1", "--cache-dtype", "fp4"])


def test_a_sequence_taken_back_gives_back_its_pages():
    c = make()
    s = c.acquire()
    c.reserve(s, 130)
    c.set_length(s, 130)
    free = c.free_pages()
    kept = c.group_of[0].pages[s][:2]
    c.rewind(s, 128)
    assert c.length(s) == 128 and c.group_of[0].pages[s] == kept
    assert c.free_pages()[0] == free[0] + 1
    assert c.group_of[0].table_flat([s], 3) == kept + [-1]
    c.reserve(s, 200)
    assert len(c.group_of[0].pages[s]) == 4
    c.set_length(s, 140)
    c.rewind(s, 140)
    c.rewind(s, 129)
    for bad in (130, -1):
        with pytest.raises(CacheError, match="taken back"):
            c.rewind(s, bad)
    c.release(s)
    assert c.free_pages() == [g.n_pages for g in c.groups]
    with pytest.raises(CacheError):
        c.rewind(s, 0)


def test_a_ring_that_has_written_over_what_is_needed_refuses():
    c = make(step_tokens=10)                                  # rings of 128 for windows of 70
    g = c.group_of[1]
    assert g.ring == 128
    s = c.acquire()
    c.reserve(s, 300)
    for end in (127, 128, 129, 200, 300):
        c.set_length(s, end)
        for length in range(end + 1):
            # the place of every position that the next token, at ``length``, sees
            seen = range(max(0, length - 69), length)
            holds = [p for p in seen if any(q % 128 == p % 128 for q in range(p + 1, end))]
            assert g.keeps(end, length) == (not holds), (end, length)
    c.set_length(s, 300)
    with pytest.raises(CacheError, match="ring"):
        c.rewind(s, 200)
    assert c.length(s) == 300 and len(c.group_of[0].pages[s]) == 5       # nothing was taken back
    c.rewind(s, 241)
    assert c.length(s) == 241 and len(g.pages[s]) == 2
