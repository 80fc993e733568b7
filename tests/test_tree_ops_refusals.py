"""What tree_attn, block_tables, tree_commit and qkv_rope_append_at refuse, without a GPU: shapes, types and strides by the
Python layer, sizes and alignments by the C entry points before any launch."""

import pytest
import torch

from quic_cu_b200 import kernels as K

I32 = dict(dtype=torch.int32)


def _attention(**more):
    a = dict(q=torch.zeros(4, 14, 64).half(), kcache=torch.zeros(3, 2, 16, 64).half(), vcache=torch.zeros(3, 2, 16, 64).half(),
             tables=torch.zeros(2, 3, **I32), lengths=torch.zeros(2, **I32), row_start=torch.zeros(3, **I32))
    a.update(more)
    return K.tree_attn(**a)


@pytest.mark.parametrize("more,match", [
    ({}, "CUDA tensors"),
    (dict(q=torch.zeros(4, 14, 64)), "one type"),
    (dict(q=torch.zeros(4, 14, 64).bfloat16()), "one type"),
    (dict(vcache=torch.zeros(3, 2, 16, 64).bfloat16()), "one type"),
    (dict(vcache=torch.zeros(3, 2, 8, 64).half()), "expected q"),
    (dict(q=torch.zeros(4, 14 * 64).half()), "expected q"),
    (dict(q=torch.zeros(4, 14, 32).half()), "head dimension"),
    (dict(q=torch.zeros(4, 15, 64).half()), "multiple of the KV heads"),
    (dict(q=torch.zeros(4, 14, 128).half()[:, :, ::2]), "contiguous"),
    (dict(kcache=torch.zeros(3, 2, 64, 16).half().transpose(2, 3)), "contiguous"),
    (dict(tables=torch.zeros(2, 6, **I32)[:, ::2]), "contiguous"),
    (dict(tables=torch.zeros(2, 3).long()), "int32"),
    (dict(lengths=torch.zeros(2)), "int32"),
    (dict(lengths=torch.zeros(3, **I32)), "requests"),
    (dict(row_start=torch.zeros(2, **I32)), "requests"),
    (dict(mask=torch.zeros(4, 1).bool()), "int32"),
    (dict(mask=torch.zeros(3, 1, **I32)), "mask must be"),
    (dict(mask=torch.zeros(4, 0, **I32)), "mask must be"),
])
def test_attention_refuses(more, match):
    with pytest.raises(RuntimeError, match=match):
        _attention(**more)


def _tables(**more):
    a = dict(tables=torch.zeros(2, 3, **I32), held=torch.zeros(2, **I32), pool=K.block_pool(5, "cpu"), lengths=torch.zeros(2, **I32),
             n_new=torch.zeros(2, **I32), block_size=16, max_rows=4)
    a.update(more)
    return K.block_tables(**a)


@pytest.mark.parametrize("more,match", [
    ({}, "CUDA tensors"),
    (dict(held=torch.zeros(2).long()), "int32"),
    
    (dict(parents=torch.zeros(4).long()), "int32"),
    (dict(parents=torch.zeros(3, 1, **I32)), "parents"),
    (dict(tables=torch.zeros(2, 0, **I32)), "tables must be"),
    (dict(tables=torch.zeros(3, **I32)), "tables must be"),
    (dict(tables=torch.zeros(3, **I32).expand(2, 3)), "tables must be"),
    (dict(lengths=torch.zeros(3, **I32)), "requests"),
    (dict(n_new=torch.zeros(4, **I32)[::2]), "contiguous"),
    (dict(pool=torch.zeros(3, **I32)), "pool"),
    (dict(max_rows=-1), "max_rows"),
])
def test_tables_refuse(more, match):
    with pytest.raises(RuntimeError, match=match):
        _tables(**more)


def test_pool():
    assert K.block_pool(3, "cpu").tolist() == [0, 3, 0, 0, 0, 1, 2]
    assert K.block_pool(4, "cpu", torch.tensor([2, 0])).tolist() == [0, 2, 0, 0, 2, 0, 0, 0]
    with pytest.raises(RuntimeError, match="more free blocks"):
        K.block_pool(1, "cpu", torch.tensor([0, 1]))


def _commit(**more):
    a = dict(kv=torch.zeros(1, 2, 3, 2, 16, 64).half(), tables=torch.zeros(2, 3, **I32), lengths=torch.zeros(2, **I32),
             row_start=torch.zeros(3, **I32), parents=torch.zeros(4, **I32), tokens=torch.zeros(4, **I32),
             targets=torch.zeros(4, **I32), max_new=4)
    a.update(more)
    return K.tree_commit(**a)


@pytest.mark.parametrize("more,match", [
    ({}, "CUDA tensors"),
    (dict(kv=torch.zeros(1, 2, 3, 2, 16, 64)), "2-byte"),
    (dict(kv=torch.zeros(2, 3, 2, 16, 64).half()), "kv must be"),
    (dict(kv=torch.zeros(1, 2, 3, 2, 64, 16).half().transpose(4, 5)), "contiguous"),
    (dict(kv=torch.zeros(1, 2, 0, 2, 16, 64).half()), "no blocks"),
    (dict(tokens=torch.zeros(4).long()), "must both be int32 or both int64"),
    (dict(targets=torch.zeros(5, **I32)), "do not match"),
    (dict(parents=torch.zeros(4).long()), "int32"),
    (dict(row_start=torch.zeros(4, **I32)), "do not match"),
])
def test_commit_refuses(more, match):
    with pytest.raises(RuntimeError, match=match):
        _commit(**more)


def test_append_refuses():
    a = dict(qkv=torch.zeros(2, 1152).half(), slot_map=torch.zeros(2).long(), positions=torch.zeros(2, **I32),
             cos=torch.zeros(8, 32).half(), sin=torch.zeros(8, 32).half(), kcache=torch.zeros(3, 2, 16, 64).half(),
             vcache=torch.zeros(3, 2, 16, 64).half())
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        K.qkv_rope_append_at(**a)
    assert K.lib().quic_qkv_rope_append_at(*[None] * 5, 8, *[None] * 3, 16, 3, 2, None) == -1


def _call(**more):
    """quic_tree_attn with made-up addresses: every refusal comes before the first of them is used."""
    a = dict(q=4096, k=4096, v=4096, out=4096, q_row=896, q_head=64, k_block=2048, k_head=1024, k_tok=64, v_block=2048, v_head=1024,
             v_tok=64, tables=4096, table_row=3, lengths=4096, row_start=4096, mask=0, mask_row=0, mask_words=0, rows=4, requests=2,
             heads=14, kv_heads=2, dim=64, n_blocks=3, block_size=16, max_blocks=3, dtype=0, max_new=4, max_len=40, scale=-1.0)
    a.update(more)
    rc = K.lib().quic_tree_attn(K._TREE_ATTN.pack(*a.values()), None, None)
    return rc, K.lib().quic_last_error().decode()


@pytest.mark.parametrize("more,code", [
    (dict(dtype=2), -2), (dict(dim=96), -2), (dict(heads=15), -2), (dict(rows=-1), -2), (dict(n_blocks=0), -2), (dict(block_size=0), -2),
    (dict(max_blocks=0), -2), (dict(block_size=1 << 16, max_blocks=1 << 14), -2), (dict(max_new=0), -2), (dict(max_len=-1), -2),
    (dict(q=0), -1), (dict(tables=0), -1), (dict(mask=4096), -2), (dict(q=4104), -1), (dict(k_tok=68), -1), (dict(q_row=900), -1),
    (dict(requests=70000), -4), (dict(rows=1 << 28, heads=14), -4), (dict(max_len=100000, block_size=4096, max_blocks=100), -1)])
def test_attention_entry_point_refuses(more, code):
    rc, message = _call(**more)
    assert rc == code and "tree_attn" in message


def test_nothing_to_do_is_no_error():
    assert _call(rows=0)[0] == 0 and _call(requests=0)[0] == 0


def test_attention_scratch():
    size = K.lib().quic_tree_attn_scratch_bytes
    assert size(1, 14, 2, 64, 1, 64) >= 2 * 148 * 32 * 66 * 4  # (two parts of 32 rows a CTA of the tcgen05 form)
    assert size(1, 14, 2, 64, 64, 8192) >= 2 * 148 * 256 * 66 * 4 > size(1, 14, 2, 64, 1, 8192)
    assert size(1, 15, 2, 64, 1, 8192) == 0 and size(0, 14, 2, 64, 1, 8192) == 0 and size(1, 14, 2, 96, 1, 8192) == 0


def test_commit_entry_point_refuses():
    names = [n for n in ("kv kv_layer kv_kind kv_block kv_head kv_tok tables table_row lengths row_start parents tokens targets token_bytes "
                         "layers n_blocks kv_heads block_size dim max_blocks rows requests max_new path accepted next_token new_lengths").split()]
    good = dict(zip(names, [4096, 12288, 6144, 2048, 1024, 64, 4096, 3, 4096, 4096, 4096, 4096, 4096, 4, 1, 3, 2, 16, 64, 3, 4, 2, 4,
                            4096, 4096, 4096, 8192]))
    for more, code in ((dict(token_bytes=2), -2), (dict(dim=12), -2), (dict(max_new=1025), -4), (dict(max_new=0), -4), (dict(kv=4100), -1),
                       (dict(kv_tok=65), -1), (dict(new_lengths=4096), -1), (dict(path=0), -1), (dict(requests=70000), -4)):
        assert K.lib().quic_tree_commit(K._TREE_COMMIT.pack(*{**good, **more}.values()), None) == code, more


def test_tables_entry_point_refuses():
    def call(requests=2, block=16, max_rows=4, n_blocks=5, max_blocks=3, parents=0, words=0, tables=4096):
        values = (tables, 3, 4096, 4096, 4096, 4096, parents, 4096, 4096, 4096, 0, max_blocks, n_blocks, requests, block, 4, words, max_rows)
        return K.lib().quic_block_tables(K._BLOCK_TABLES.pack(*values), None)
    assert call(tables=0) == -1 and call(parents=4096) == -1 and call(parents=4096, words=1) == -1
    assert call(requests=0) == -2 and call(block=0) == -2 and call(max_blocks=0) == -2 and call(n_blocks=-1) == -2
    assert call(requests=4097) == -4 and call(max_rows=1 << 25) == -4 and call(block=1 << 20, max_blocks=1 << 10) == -2
