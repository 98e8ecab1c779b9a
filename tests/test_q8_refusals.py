"""What the 8-bit cache's operators and the verification of drafted tokens refuse, before anything is launched
(no GPU needed)."""
import pytest
import torch

from minfer_b200.kernels import api as K

I32 = torch.int32


def pages(n=3, kv=2, dim=64, dtype=torch.int8, **change):
    return K.q8_pages(n, kv, dim, dtype, device="cpu")._replace(**change)


def attend(**change):
    a = dict(q=torch.zeros(4, 6, 64), pages=pages(), cu_seqlens=torch.tensor([0, 1, 4], dtype=I32),
             seq_end=torch.tensor([5, 9], dtype=I32), page_table=torch.zeros(2, 1, dtype=I32), table_stride=1, ring=0,
             out=torch.zeros(4, 6, 64), max_row_tokens=3, max_end=9, n_heads=6, n_kv=2, head_dim=64, window=0,
             scale=0.1, status=torch.zeros(1, dtype=I32))
    a.update(change)
    K.attention_paged_q8(**a)


def store(**change):
    a = dict(qkv=torch.zeros(4, 10 * 64), positions=torch.zeros(4, dtype=I32), token_row=torch.zeros(4, dtype=I32),
             seq_end=torch.tensor([5, 9], dtype=I32), inv_freq=torch.zeros(32, dtype=torch.float64),
             q_out=torch.zeros(4, 6, 64), k_out=torch.zeros(4, 2, 64), v_out=torch.zeros(4, 2, 64), pages=pages(),
             page_table=torch.zeros(2, 1, dtype=I32), table_stride=1, ring=0, n_heads=6, n_kv=2, head_dim=64,
             rotary_dim=64, style=0, status=torch.zeros(1, dtype=I32))
    a.update(change)
    K.rope_kvstore_q8(**a)


def read(**change):
    a = dict(pages=pages(), page_table=torch.zeros(2, 1, dtype=I32), table_stride=1, ring=0,
             seq_end=torch.tensor([5, 9], dtype=I32), k_out=torch.zeros(2, 2, 64, 64), v_out=torch.zeros(2, 2, 64, 64),
             status=torch.zeros(1, dtype=I32))
    a.update(change)
    K.read_pages_q8(**a)


def verify(**change):
    a = dict(logits=torch.zeros(5, 10), drafts=torch.zeros(3, dtype=I32), cu_drafts=torch.tensor([0, 1, 3], dtype=I32),
             draft_logits=torch.zeros(3, 10), accept_u=torch.zeros(3), draw_u=torch.zeros(2), temperature=1.0,
             accepted=torch.zeros(2, dtype=I32), tokens=torch.zeros(2, dtype=I32))
    a.update(change)
    K.verify_drafts(**a)


def test_nothing_runs_on_the_cpu():
    for call in (attend, store, read, verify):
        with pytest.raises(K.KernelError, match="CUDA device"):
            call()


@pytest.mark.parametrize("change,why", [
    (dict(n_heads=5), "do not divide"),
    (dict(pages=pages(dim=128)), "pages must be"),
    (dict(pages=pages(kv=1)), "pages must be"),
    (dict(pages=pages(k=torch.zeros(3, 2, 64, 64))), "float8_e4m3fn or int8"),
    (dict(pages=pages(v=torch.zeros(3, 2, 64, 64, dtype=torch.int8).view(torch.float8_e4m3fn))), "alike"),
    (dict(pages=pages(k_scale=torch.zeros(3, 2, 63))), "a scale belongs"),
    (dict(pages=pages(v_scale=torch.zeros(3, 2, 64, dtype=torch.bfloat16))), "float32"),
    (dict(q=torch.zeros(4, 5, 64)), "q and out"),
    (dict(out=torch.zeros(4, 6, 64, dtype=torch.bfloat16)), "q and out"),
    (dict(cu_seqlens=torch.zeros(2, dtype=I32)), "cu_seqlens"),
    (dict(window=-1), "ring"),
    (dict(ring=63, window=3), "ring"),
    (dict(ring=64), "ring"),
    (dict(ring=64, window=63), "ring"),               # 3 new tokens: the first one's window is overwritten
    (dict(scale=float("nan")), "finite"),
    (dict(table_stride=2), "page table"),
    (dict(table_stride=0), "page table"),
])
def test_attention_refuses(change, why):
    with pytest.raises(K.KernelError, match=why):
        attend(**change)


@pytest.mark.parametrize("change,why", [
    (dict(qkv=torch.zeros(4, 9 * 64)), "width"),
    (dict(n_partials=2), "splits"),
    (dict(qkv=torch.zeros(2, 4, 640)), "tokens, width"),
    (dict(bias=torch.zeros(7)), "bias"),
    (dict(q_out=torch.zeros(4, 5, 64)), "q has"),
    (dict(k_out=torch.zeros(4, 2, 64, dtype=torch.bfloat16)), "keys and values"),
    (dict(v_out=torch.zeros(3, 2, 64)), "keys and values"),
    (dict(positions=torch.zeros(3, dtype=I32)), "position"),
    (dict(rotary_dim=32), "frequencies"),
    (dict(ring=1), "ring"),
    (dict(table_stride=5), "page table"),
    (dict(pages=pages(dim=32)), "pages must be"),
])
def test_store_refuses(change, why):
    with pytest.raises(K.KernelError, match=why):
        store(**change)


@pytest.mark.parametrize("change,why", [
    (dict(k_out=torch.zeros(1, 2, 64, 64)), "outputs"),
    (dict(v_out=torch.zeros(2, 2, 64, 64, dtype=torch.bfloat16)), "one type"),
    (dict(ring=-64), "ring"),
    (dict(table_stride=3), "page table"),
    (dict(pages=pages(k_scale=torch.zeros(2, 2, 64))), "a scale belongs"),
])
def test_read_refuses(change, why):
    with pytest.raises(K.KernelError, match=why):
        read(**change)


@pytest.mark.parametrize("change,why", [
    (dict(logits=torch.zeros(5, 10, dtype=torch.bfloat16)), "float32 rows"),
    (dict(logits=torch.zeros(10, 5).t()), "contiguous"),
    (dict(logits=torch.zeros(4, 10)), "rows of logits"),
    (dict(draft_logits=torch.zeros(3, 11)), "drafts' logits"),
    (dict(draft_logits=torch.zeros(3, 10, dtype=torch.float64)), "drafts' logits"),
    (dict(draft_logits=torch.zeros(10, 3).t()), "drafts' logits"),
    (dict(accept_u=torch.zeros(2)), "sizes"),
    (dict(cu_drafts=torch.zeros(2, dtype=I32)), "sizes"),
    (dict(tokens=torch.zeros(3, dtype=I32)), "sizes"),
    (dict(temperature=-0.1), "temperature"),
    (dict(temperature=float("inf")), "temperature"),
    (dict(temperature=2e30), "temperature"),
    (dict(temperature=float("nan")), "temperature"),
])
def test_verify_refuses(change, why):
    with pytest.raises(K.KernelError, match=why):
        verify(**change)


def test_pages_are_made_in_two_formats():
    for dtype in (torch.int8, torch.float8_e4m3fn):
        p = K.q8_pages(2, 3, 32, dtype, device="cpu")
        assert p.k.dtype == p.v.dtype == dtype and p.k.shape == (2, 3, 64, 32) and p.k_scale.shape == (2, 3, 64)
        assert not p.k.float().any() and not p.v_scale.any() and p.k.data_ptr() != p.v.data_ptr()
    with pytest.raises(K.KernelError, match="float8_e4m3fn or int8"):
        K.q8_pages(1, 1, 16, torch.bfloat16, device="cpu")
