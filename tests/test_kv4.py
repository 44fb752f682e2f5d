"""CPU tests of the 4-bit cache's host side: argument checks of the Python calls and of the C ABI (nothing is launched),
the C structures' layout, the oracle's own byte layout and quantiser."""
import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as ora

REPO = Path(__file__).resolve().parent.parent


def test_ctypes_layout_matches_header(tmp_path):
    from tilemix_b200._lib import TmBlockTablesParams, TmKv4AttnParams

    structs = {"tm_block_tables_params": TmBlockTablesParams, "tm_kv4_attn_params": TmKv4AttnParams}
    src = ["#include <stdio.h>", "#include <stddef.h>", '#include "tilemix_b200.h"', "int main(void) {"]
    for name, cls in structs.items():
        src.append(f'printf("{name} %zu\\n", sizeof({name}));')
        src += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, *_ in cls._fields_]
    (tmp_path / "layout.c").write_text("\n".join(src + ["return 0; }"]))
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")],
                   check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = dict(line.rsplit(" ", 1) for line in out.splitlines())
    for name, cls in structs.items():
        assert int(got[name]) == ctypes.sizeof(cls)
        for f, *_ in cls._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(cls, f).offset, (name, f)


@pytest.mark.parametrize("dim", [64, 128])
def test_block_layout_covers_every_byte_once(dim):
    """The 16 tokens' codes, scales and minima fill a block of 20 dim bytes without overlap."""
    used = np.zeros(20 * dim, dtype=int)
    for tok in range(16):
        kc, vc, ks, vs = ora.block_offsets(dim, tok)
        for codes in (kc, vc):
            np.add.at(used, codes[0::2], 1)
            assert np.array_equal(codes[0::2], codes[1::2])
        for scales, low in ((ks, 2), (vs, 8)):
            for byte in (0, 1):
                np.add.at(used, scales + byte, 1)
                np.add.at(used, scales + low + byte, 1)
    assert (used == 1).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_oracle_round_trip(dim):
    """Half a step: a value reads back within scale / 2 of what was stored, plus what rounding the scale down takes from 15
    codes (at most 2^-10 each)."""
    rng = np.random.default_rng(dim)
    k, v = (rng.standard_normal((21, 3, dim)).astype(np.float16) for _ in range(2))
    pool = np.zeros((2, 3, 2 * 20 * dim), dtype=np.uint8)
    slots = np.concatenate([rng.permutation(64)[:20], [-1]])
    ora.append(pool, k, v, slots)
    for x, got in zip((k, v), ora.read(pool, slots, dim)):
        _, scale, _ = ora.quantise(x)
        step = np.repeat(scale.astype(np.float64), 32, axis=-1).reshape(x.shape)
        assert (np.abs(got - x.astype(np.float64))[:20] <= (step * (0.5 + 15 * 2.0 ** -10))[:20]).all()
        assert (got[20] == 0).all()


class _Fake:
    """The attributes that the argument checks read (no device needed)."""

    def __init__(self, shape, dtype=torch.float16, device="cuda:0", stride=None, is_cuda=True):
        self.shape, self.dtype, self.device, self.is_cuda = torch.Size(shape), dtype, torch.device(device), is_cuda
        self.ndim, self._stride = len(shape), stride
        if stride is None:
            self._stride = [int(np.prod(shape[i + 1:])) for i in range(len(shape))]

    def numel(self):
        return int(np.prod(self.shape))

    def get_device(self):
        return self.device.index if self.is_cuda else -1

    def stride(self, i=None):
        return tuple(self._stride) if i is None else self._stride[i]

    def new_empty(self, *shape):
        raise AssertionError("an argument check is missing: the call went on to allocate")

    def is_contiguous(self):
        return list(self._stride) == [int(np.prod(self.shape[i + 1:])) for i in range(self.ndim)]


def _pool(pages=4, heads=2, page_size=32, dim=64, **over):
    return _Fake((pages, heads, page_size // 16 * 20 * dim), over.pop("dtype", torch.uint8), **over)


def _i32(*shape, **over):
    return _Fake(shape, over.pop("dtype", torch.int32), **over)


ATTN = dict(q=lambda: _Fake((3, 4, 64)), pool=_pool, block_table=lambda: _i32(3, 5), kv_lens=lambda: _i32(3))


@pytest.mark.parametrize("change,exc,text", [
    (dict(q=_Fake((3, 4, 64), is_cuda=False)), RuntimeError, "CUDA kernel"),
    (dict(q=_Fake((3, 4))), ValueError, "expected q"),
    (dict(q=_Fake((3, 4, 64), torch.bfloat16)), TypeError, "float16"),
    (dict(q=_Fake((3, 4, 96))), ValueError, "head_dim"),
    (dict(q=_Fake((3, 3, 64))), ValueError, "divisible"),
    (dict(q=_Fake((3, 4, 64), stride=(512, 128, 2))), ValueError, "contiguous"),
    (dict(q=_Fake((4, 4, 64))), ValueError, "one query row"),
    (dict(max_seqlen_q=2), ValueError, "one query row"),
    (dict(max_seqlen_q=0, cu_seqlens_q=_i32(4)), ValueError, "positive"),
    (dict(pool=_pool(dtype=torch.int8)), TypeError, "uint8"),
    (dict(pool=_Fake((4, 2, 100), torch.uint8)), ValueError, "whole blocks"),
    (dict(pool=_pool(device="cuda:1")), ValueError, "one CUDA device"),
    (dict(block_table=_i32(3, 5, dtype=torch.int64)), TypeError, "int32"),
    (dict(block_table=_i32(3, 5, stride=(10, 2))), ValueError, "contiguous"),
    (dict(kv_lens=_i32(2)), ValueError, "batch"),
    (dict(cu_seqlens_q=_i32(3)), ValueError, "batch \\+ 1"),
    (dict(key_mask=_i32(3, 9)), TypeError, "bool"),
    (dict(key_mask=_i32(2, 9, dtype=torch.bool)), ValueError, "row for each"),
    (dict(out=_Fake((3, 4, 128)), sm_scale=1.0), ValueError, "match q"),
    (dict(out=_Fake((3, 4, 64)), sm_scale=0.0), ValueError, "sm_scale"),
    (dict(out=_Fake((3, 4, 64)), sm_scale=float("nan")), ValueError, "sm_scale"),
])
def test_attention_refusals(change, exc, text):
    from tilemix_b200.attention.kv4 import kv4_attention

    args = {name: make() for name, make in ATTN.items()}
    args.update(change)
    with pytest.raises(exc, match=text):
        kv4_attention(**args)


@pytest.mark.parametrize("change,exc,text", [
    (dict(k=_Fake((6, 2, 64), is_cuda=False)), RuntimeError, "CUDA kernel"),
    (dict(v=_Fake((6, 1, 64))), ValueError, "shapes"),
    (dict(k=_Fake((6, 2))), ValueError, "expected"),
    (dict(v=_Fake((6, 2, 64), torch.float32)), TypeError, "float16"),
    (dict(v=_Fake((6, 2, 64), device="cuda:1")), ValueError, "one CUDA device"),
    (dict(pool=_pool(heads=3)), ValueError, "KV heads"),
    (dict(slots=_Fake((6,), torch.int32)), TypeError, "int64"),
    (dict(slots=_Fake((5,), torch.int64)), ValueError, "5 slots for 6"),
    (dict(k=_Fake((6, 2, 64), stride=(256, 128, 2))), ValueError, "contiguous"),
])
def test_append_refusals(change, exc, text):
    from tilemix_b200.attention.kv4 import kv4_append

    args = dict(k=_Fake((6, 2, 64)), v=_Fake((6, 2, 64)), pool=_pool(), slots=_Fake((6,), torch.int64))
    args.update(change)
    with pytest.raises(exc, match=text):
        kv4_append(**args)


@pytest.mark.parametrize("change,exc,text", [
    (dict(cached_lens=_i32(3, is_cuda=False)), RuntimeError, "CUDA kernel"),
    (dict(cached_lens=_i32(3, dtype=torch.int64)), TypeError, "int32"),
    (dict(new_lens=_i32(2)), ValueError, "batch"),
    (dict(block_table=_i32(3)), ValueError, "2 dimensions"),
    (dict(free_span=_i32(2)), TypeError, "int64"),
    (dict(free_span=_Fake((3,), torch.int64)), ValueError, "two entries"),
    (dict(page_size=24), ValueError, "multiple of 16"),
    (dict(page_size=0), ValueError, "multiple of 16"),
    (dict(max_new_tokens=-1), ValueError, "max_new_tokens"),
    (dict(cached_lens=_i32(8193), new_lens=_i32(8193), block_table=_i32(8193, 5)), ValueError, "8192"),
])
def test_table_refusals(change, exc, text):
    from tilemix_b200.attention.kv4 import build_block_tables

    args = dict(cached_lens=_i32(3), new_lens=_i32(3), block_table=_i32(3, 5), free_pages=_i32(16),
                free_span=_Fake((2,), torch.int64), page_size=32, max_new_tokens=8)
    args.update(change)
    with pytest.raises(exc, match=text):
        build_block_tables(**args)


def test_pool_and_release_refusals():
    from tilemix_b200.attention.kv4 import kv4_pool, kv4_read, release_pages

    for bad in (dict(head_dim=80), dict(page_size=8), dict(kv_heads=0), dict(num_pages=-1)):
        args = dict(num_pages=2, page_size=16, kv_heads=1, head_dim=64)
        args.update(bad)
        with pytest.raises(ValueError):
            kv4_pool(**args, device="cpu")
    pool = kv4_pool(2, 16, 1, 64, device="cpu")
    assert pool.shape == (2, 1, 1280)
    with pytest.raises(RuntimeError):
        kv4_read(pool, torch.zeros(1, dtype=torch.int64), 64)
    with pytest.raises(TypeError, match="bool"):
        release_pages(_i32(3), _i32(3), _i32(3, 5), _i32(16), _Fake((2,), torch.int64), page_size=16)


def test_c_abi_refusals_need_no_gpu():
    """Statuses of the C entry points for arguments that are refused on the host."""
    from tilemix_b200._lib import TmBlockTablesParams, TmKv4AttnParams, lib

    fake = 0x100000
    need = ctypes.c_int64()

    def attn(**over):
        p = TmKv4AttnParams()
        for name in ("q", "out", "pool", "block_table", "kv_lens"):
            setattr(p, name, fake)
        p.q_stride_tok = p.o_stride_tok = 8 * 128
        p.q_stride_head = p.o_stride_head = 128
        p.q_tokens = p.batch = 4
        p.num_pages, p.table_stride, p.cols, p.page_size = 16, 4, 4, 32
        p.heads_q, p.heads_k, p.head_dim, p.max_seqlen_q, p.max_kv_len, p.causal, p.sm_scale = 8, 2, 128, 1, 128, 1, 0.1
        for k, v in over.items():
            setattr(p, k, v)
        return lib().tm_kv4_attn_workspace(ctypes.addressof(p), ctypes.byref(need)), p

    assert attn()[0] == 0
    for status, over in ((-1, dict(q=None)), (-1, dict(kv_lens=None)), (-1, dict(pool=None)), (-2, dict(heads_q=7)),
                         (-2, dict(page_size=24)), (-2, dict(page_size=0)), (-4, dict(head_dim=96)),
                         (-4, dict(batch=65536)), (-2, dict(max_seqlen_q=2)), (-3, dict(q=fake + 8)),
                         (-3, dict(q_stride_head=132)), (-3, dict(pool=fake + 8)), (-4, dict(max_kv_len=2**30 + 1)),
                         (-2, dict(q_tokens=3)), (-2, dict(sm_scale=0.0)), (-2, dict(sm_scale=float("inf")))):
        assert attn(**over)[0] == status, over
    assert lib().tm_kv4_attn_workspace(None, ctypes.byref(need)) == -1
    assert attn(q_tokens=2**31, max_seqlen_q=65535, cu_seqlens_q=fake, max_kv_len=2**30, cols=2**25)[0] == -4
    # the parts of a split key axis need their workspace
    rc, p = attn(batch=1, q_tokens=1, max_kv_len=1 << 20, cols=1 << 15)
    assert rc == 0 and need.value > 0
    assert lib().tm_kv4_attn(ctypes.addressof(p), None, 0, None, None) == -1
    assert lib().tm_kv4_attn(ctypes.addressof(p), fake, need.value - 1, None, None) == -2
    assert lib().tm_kv4_attn(ctypes.addressof(p), fake + 4, need.value, None, None) == -3

    args = [fake, 256, 128, fake, 256, 128, 4, fake, fake, 8, 2, 128, 32, None, None]
    for at, value, status in ((0, None, -1), (7, None, -1), (8, None, -1), (0, fake + 2, -3), (1, 260, -3),
                              (10, 0, -2), (11, 32, -4), (12, 20, -2), (6, -1, -2)):
        bad = list(args)
        bad[at] = value
        assert lib().tm_kv4_append(*bad) == status, (at, value)
    args = [fake, 8, 2, 128, 32, fake, 4, fake, fake, None, None]
    for at, value, status in ((0, None, -1), (5, None, -1), (7, None, -1), (7, fake + 2, -3), (2, 0, -2), (3, 32, -4)):
        bad = list(args)
        bad[at] = value
        assert lib().tm_kv4_read(*bad) == status, (at, value)

    def tables(**over):
        p = TmBlockTablesParams()
        for i, name in enumerate(("cached_lens", "new_lens", "block_table", "free_pages", "free_span", "slots",
                                  "positions", "cu_seqlens", "kv_lens", "free_span_out")):
            setattr(p, name, fake + 4096 * i)
        p.table_stride, p.cols, p.capacity, p.batch, p.page_size, p.n_slots = 4, 4, 8, 3, 16, 5
        for k, v in over.items():
            setattr(p, k, v)
        return lib().tm_build_block_tables(ctypes.addressof(p), None, None)

    for status, over in ((-1, dict(free_span=None)), (-1, dict(slots=None)), (-1, dict(kv_lens=None)),
                         (-2, dict(page_size=8)), (-2, dict(n_slots=-1)), (-4, dict(batch=8193)),
                         (-4, dict(kv_lens=fake)), (-4, dict(free_span_out=fake + 4096 * 4))):
        assert tables(**over) == status, over
    assert lib().tm_release_pages(None, None, None, 0, 4, None, 8, None, 3, 16, None, None) == -1
    assert lib().tm_release_pages(fake, fake, fake, 4, 4, fake, 8, fake, 3, 17, None, None) == -2


def test_the_first_call_cannot_be_captured(monkeypatch):
    """It allocates the error word, which must not belong to a graph's memory."""
    from tilemix_b200 import _lib
    from tilemix_b200.attention import tilemix

    monkeypatch.setattr(_lib, "_ERROR_WORD_PTRS", {})
    monkeypatch.setattr(tilemix, "_ERROR_WORDS", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before the capture"):
        _lib.error_word_ptr(0)


def test_token_counts_stay_clear_of_32_bits():
    """The grid counts 16 tokens a CTA in two of its dimensions, the last rounded up to whole 65,535 CTAs: up to 2^20 tokens
    more than there are, all of them below 2^31."""
    from tilemix_b200._lib import lib

    fake = 0x100000
    for tokens in (2**31 - 17, 2**31 - 2**20):
        assert lib().tm_kv4_append(fake, 0, 64, fake, 0, 64, tokens, fake, fake, 8, 1, 64, 32, None, None) == -4
        assert lib().tm_kv4_read(fake, 8, 1, 64, 32, fake, tokens, fake, fake, None, None) == -4
    groups = (2**31 - 1 - 2**20 + 15) // 16  # of the most tokens that are taken
    assert -(-groups // 65535) * 65535 * 16 <= 2**31


def test_scales_whose_scores_leave_fp32_are_refused():
    """|q . k| is at most 128 * 65504^2 < 2^40: times log2(e) 2^80 every score is finite, times a scale of 2^127 none is."""
    from tilemix_b200._lib import TmKv4AttnParams, lib
    from tilemix_b200.attention.kv4 import kv4_attention

    p = TmKv4AttnParams()
    for name in ("q", "out", "pool", "block_table", "kv_lens"):
        setattr(p, name, 0x100000)
    p.q_stride_tok, p.q_stride_head, p.o_stride_tok, p.o_stride_head, p.q_tokens, p.batch = 1024, 128, 1024, 128, 4, 4
    p.num_pages, p.table_stride, p.cols, p.page_size = 16, 4, 4, 32
    p.heads_q, p.heads_k, p.head_dim, p.max_seqlen_q, p.max_kv_len = 8, 2, 128, 1, 128
    need = ctypes.c_int64()
    for scale, status in ((2.0 ** 80, 0), (2.0 ** 81, -2), (3e38, -2)):
        p.sm_scale = scale
        assert lib().tm_kv4_attn_workspace(ctypes.addressof(p), ctypes.byref(need)) == status, scale
        if status:
            with pytest.raises(ValueError, match="sm_scale"):
                kv4_attention(**{name: make() for name, make in ATTN.items()}, out=_Fake((3, 4, 64)), sm_scale=scale)


@pytest.mark.parametrize("columns", [2**25 + 1, 2**27])
def test_tables_of_more_than_2_30_keys(columns):
    """Such a table's capacity is no bound to plan for: keys are counted up to 2^30, and the call goes on to allocate."""
    from tilemix_b200.attention.kv4 import kv4_attention

    args = {name: make() for name, make in ATTN.items()}
    args.update(block_table=_i32(3, columns), out=_Fake((3, 4, 64)))
    with pytest.raises(AssertionError, match="went on to allocate"):
        kv4_attention(**args)


def test_threads_share_one_error_word(monkeypatch):
    """Two threads whose first calls overlap: both launch with the word that is read, and that stays allocated."""
    from tilemix_b200 import _lib
    from tilemix_b200.attention import tilemix

    monkeypatch.setattr(_lib, "_ERROR_WORD_PTRS", {})
    monkeypatch.setattr(tilemix, "_ERROR_WORDS", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    others, kept, zeros = [], [], torch.zeros

    def overlapping(*size, dtype, device):
        if not others:  # the other thread makes its whole call while this one allocates
            others.append(None)
            others[0] = _lib.error_word_ptr(0)
        kept.append(zeros(*size, dtype=dtype))
        return kept[-1]

    monkeypatch.setattr(torch, "zeros", overlapping)
    mine = _lib.error_word_ptr(0)
    assert mine == others[0] == _lib.error_word_ptr(0) == tilemix._ERROR_WORDS[0].data_ptr()
