"""GPU tests of the paged 4-bit cache and the attention over it against the numpy oracle: integers and stored bytes
exactly, attention within the oracle's derived rounding bound."""
import numpy as np
import pytest
import torch

from oracle import kv4_oracle as ora

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error():
    from tilemix_b200.attention.tilemix import device_error_code

    if torch.cuda.is_available():
        device_error_code()
    yield
    if torch.cuda.is_available():
        assert device_error_code() == 0


def _error_code():
    from tilemix_b200.attention.tilemix import device_error_code

    return device_error_code()


# ---------------------------------------------------------------------------------------------- block tables
def _tables_case(cached, new, page, seed, extra_pages=5, extra_cols=2, head=None):
    rng = np.random.default_rng(seed)
    cached, new = np.asarray(cached), np.asarray(new)
    held, total = -(-cached // page), -(-(cached + new) // page)
    capacity = int(total.sum()) + extra_pages
    order = rng.permutation(capacity).astype(np.int32)
    table = np.full((len(cached), int(total.max(initial=0)) + extra_cols), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    head = int(rng.integers(0, capacity)) if head is None else head
    ring = np.full(capacity, -7, dtype=np.int32)
    free = order[at:]
    ring[(head + np.arange(len(free))) % capacity] = free
    return cached, new, table, ring, np.array([head, head + len(free)], dtype=np.int64)


def _build(dev, cached, new, table, ring, span, page, rows):
    from tilemix_b200.attention.kv4 import build_block_tables

    to = lambda x, t: torch.tensor(np.asarray(x), dtype=t, device=dev)  # noqa: E731
    tab = to(table, torch.int32)
    got = build_block_tables(to(cached, torch.int32), to(new, torch.int32), tab, to(ring, torch.int32),
                             to(span, torch.int64), page_size=page, max_new_tokens=rows)
    return [x.cpu().numpy() for x in got] + [tab.cpu().numpy()]


@pytest.mark.parametrize("cached,new,page,more", [
    ([0], [1], 16, 0),
    ([15, 16, 17, 0], [1, 1, 0, 40], 16, 3),
    ([0, 0, 0], [0, 0, 0], 64, 4),
    ([5, 100, 31], [700, 0, 33], 32, 0),
    (list(range(300)), [1] * 300, 48, 7),
    ([3] * 8192, [1, 0] * 4096, 16, 1),
    ([0, 1], [70001, 5], 128, 0),
    ([], [], 16, 2),
])
def test_block_tables_match_the_oracle(cuda_device, cached, new, page, more):
    case = _tables_case(cached, new, page, seed=len(cached))
    rows = int(np.sum(new)) + more
    got, ref = _build(cuda_device, *case, page, rows), ora.build_block_tables(*case, page, rows)
    for g, r in zip(got, ref[:6]):
        assert np.array_equal(g, r)


@pytest.mark.parametrize("why", ["pages", "columns", "slots", "negative", "huge"])
def test_block_tables_allocate_all_or_nothing(cuda_device, why):
    cached, new, table, ring, span = _tables_case([10, 20, 30], [30, 1, 40], 16, seed=3, extra_pages=0, head=2)
    rows = 71
    if why == "pages":
        span[1] -= 1
    elif why == "columns":
        table = table[:, :4]
    elif why == "slots":
        rows = 70
    elif why == "negative":
        new[1] = -1
    else:
        new[1] = 2**31 - 5
    got = _build(cuda_device, cached, new, table, ring, span, 16, rows)
    assert _error_code() == 11
    assert (got[0] == -1).all() and (got[1] == 0).all() and (got[2] == 0).all()
    assert np.array_equal(got[3], cached) and np.array_equal(got[4], span) and np.array_equal(got[5], table)


def test_pages_go_round_the_ring(cuda_device):
    """Steps of growth and release keep every page in one place: in a request's row or in the ring's free part."""
    from tilemix_b200.attention.kv4 import build_block_tables, release_pages

    dev, page, pages, batch = cuda_device, 16, 40, 5
    ring = torch.randperm(pages, generator=torch.Generator().manual_seed(0)).int().to(dev)
    span = torch.tensor([0, pages], device=dev)
    table = torch.full((batch, 12), -1, dtype=torch.int32, device=dev)
    lens = torch.zeros(batch, dtype=torch.int32, device=dev)
    rng = np.random.default_rng(1)
    for step in range(40):
        new = torch.tensor(rng.integers(0, 20, batch), dtype=torch.int32, device=dev)
        t = build_block_tables(lens, new, table, ring, span, page_size=page, max_new_tokens=100)
        lens, span = t.kv_lens, t.free_span
        _error_code()  # a step that did not fit allocated nothing
        slots = t.slots[:int(t.cu_seqlens_q[-1])].cpu().numpy()
        assert len(set(slots)) == len(slots)
        done = torch.tensor(rng.random(batch) < 0.3, device=dev)
        release_pages(lens, done, table, ring, span, page_size=page)
        held = table.cpu().numpy()
        mine = held[held >= 0].tolist()
        head, tail = span.tolist()
        free = ring.cpu().numpy()[np.arange(head, tail) % pages].tolist()
        assert sorted(mine + free) == list(range(pages))
        assert ((held >= 0).sum(1) == -(-lens.cpu().numpy() // page)).all()


def test_release_refuses_an_overfull_ring(cuda_device):
    from tilemix_b200.attention.kv4 import release_pages

    dev = cuda_device
    lens = torch.tensor([20, 5], dtype=torch.int32, device=dev)
    table = torch.tensor([[3, 4], [5, -1]], dtype=torch.int32, device=dev)
    ring, span = torch.zeros(6, dtype=torch.int32, device=dev), torch.tensor([2, 6], device=dev)
    release_pages(lens, torch.tensor([True, True], device=dev), table, ring, span, page_size=16)
    assert _error_code() == 11 and lens.tolist() == [20, 5] and span.tolist() == [2, 6]
    release_pages(lens, torch.tensor([True, False], device=dev), table, ring, span, page_size=16)
    assert lens.tolist() == [0, 5] and span.tolist() == [2, 8] and table.tolist() == [[-1, -1], [5, -1]]
    assert ring[:2].tolist() == [3, 4]


# ---------------------------------------------------------------------------------------------- append and read
def _values(rng, n, heads, dim):
    """Rows with outlier channels, constant and nearly constant groups, subnormal steps and the type's extremes."""
    x = rng.standard_normal((n, heads, dim)) * np.exp(rng.uniform(-3, 3, (n, heads, 1)))
    x[..., dim // 3] *= 30
    x = x.astype(np.float16)
    if n > 4:
        x[1, :, :32] = np.float16(0.3)
        x[2, :, :32] = np.where(np.arange(32) % 2, np.float16(2e-7), np.float16(-3e-6))
        x[3, :, 32:64] = np.where(np.arange(32) % 3, np.float16(65504), np.float16(-65504))
        x[4, :, :32] = 0
    return x


@pytest.mark.parametrize("n,heads,dim,page,pad", [(1, 1, 64, 16, 0), (1, 8, 128, 64, 0), (33, 3, 64, 48, 4),
                                                  (257, 2, 128, 32, 1), (1000, 4, 128, 256, 0)])
def test_append_stores_the_oracles_bytes(cuda_device, n, heads, dim, page, pad):
    from tilemix_b200.attention.kv4 import kv4_append, kv4_pool, kv4_read

    rng = np.random.default_rng(n)
    k, v = _values(rng, n + pad, heads, dim), _values(rng, n + pad, heads, dim)
    pages = -(-n // page) + 2
    slots = np.concatenate([rng.permutation(pages * page)[:n], [-1] * pad]).astype(np.int64)
    pool = kv4_pool(pages, page, heads, dim, cuda_device)
    fill = torch.randint(0, 256, pool.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(1))
    pool.copy_(fill)  # what a slot does not own is left as it was
    ref = fill.numpy().copy()
    ora.append(ref, k, v, slots)
    to = lambda x: torch.from_numpy(x).to(cuda_device)  # noqa: E731
    kv4_append(to(k), to(v), pool, to(slots))
    assert np.array_equal(pool.cpu().numpy(), ref)
    got = kv4_read(pool, to(slots), dim)
    for g, r in zip(got, ora.read(ref, slots, dim)):
        # one rounding of s n + m in fp32, one to fp16
        off = np.abs(g.double().cpu().numpy() - r) - (np.abs(r) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25)
        assert float(off.max()) <= 0


def test_append_takes_strided_rows_and_another_stream(cuda_device):
    """The [B, H, T, D] views that a model's projections leave, on a side stream."""
    from tilemix_b200.attention.kv4 import kv4_append, kv4_pool

    rng = np.random.default_rng(5)
    k, v = (rng.standard_normal((2, 3, 40, 64)).astype(np.float16) for _ in range(2))
    pool = kv4_pool(3, 32, 3, 64, cuda_device)
    slots = rng.permutation(96)[:80].astype(np.int64)
    ref = np.zeros(pool.shape, dtype=np.uint8)
    rows = lambda x: np.ascontiguousarray(x.transpose(0, 2, 1, 3)).reshape(80, 3, 64)  # noqa: E731
    ora.append(ref, rows(k), rows(v), slots)
    dk = torch.from_numpy(k).to(cuda_device).transpose(1, 2).flatten(0, 1)
    wide = torch.from_numpy(rows(v)).to(cuda_device)
    dv = torch.cat([wide, wide], 2)[..., 64:]
    assert not dv.is_contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv4_append(dk, dv, pool, torch.from_numpy(slots).to(cuda_device))
    torch.cuda.current_stream().wait_stream(side)
    assert np.array_equal(pool.cpu().numpy(), ref)


def test_non_finite_groups_read_back_as_nan(cuda_device):
    from tilemix_b200.attention.kv4 import kv4_append, kv4_pool, kv4_read

    k = torch.ones(3, 1, 64, dtype=torch.float16, device=cuda_device)
    v = torch.ones_like(k)
    k[0, 0, 5], k[1, 0, 40], v[2, 0, 3] = float("nan"), float("inf"), float("-inf")
    pool, slots = kv4_pool(1, 16, 1, 64, cuda_device), torch.arange(3, device=cuda_device)
    kv4_append(k, v, pool, slots)
    gk, gv = kv4_read(pool, slots, 64)
    assert gk[0, 0, :32].isnan().all() and gk[1, 0, 32:].isnan().all() and gv[2, 0, :32].isnan().all()
    assert (gk[0, 0, 32:] == 1).all() and (gk[1, 0, :32] == 1).all() and (gk[2] == 1).all() and (gv[:2] == 1).all()


def test_slots_outside_the_pool_are_skipped(cuda_device):
    from tilemix_b200.attention.kv4 import kv4_append, kv4_pool, kv4_read

    x = torch.ones(3, 1, 64, dtype=torch.float16, device=cuda_device)
    pool = kv4_pool(1, 16, 1, 64, cuda_device)
    for far in (16, -2, 2**62):
        kv4_append(x, x, pool, torch.tensor([far, -1, -1], device=cuda_device))
        assert _error_code() == 13 and not pool.any()
        k, v = kv4_read(pool, torch.tensor([-1, far, -1], device=cuda_device), 64)
        assert _error_code() == 13 and not k.any() and not v.any()


def test_misaligned_rows_are_refused(cuda_device):
    from tilemix_b200.attention.kv4 import kv4_append, kv4_attention, kv4_pool

    flat = torch.zeros(4 * 64 + 4, dtype=torch.float16, device=cuda_device)
    x, pool = flat[4:].view(4, 1, 64), kv4_pool(1, 16, 1, 64, cuda_device)
    with pytest.raises(RuntimeError, match="status -3"):
        kv4_append(x, x, pool, torch.arange(4, device=cuda_device))
    with pytest.raises(RuntimeError, match="status -3"):
        kv4_attention(x, pool, torch.zeros((4, 1), dtype=torch.int32, device=cuda_device),
                      torch.ones(4, dtype=torch.int32, device=cuda_device))


# ---------------------------------------------------------------------------------------------- attention
def _cache(dev, kv_lens, heads_k, dim, page, seed, cols=None, v_scale=1.0):
    """A pool filled through the oracle, its block table, and the 64-bit keys and values of each request."""
    rng = np.random.default_rng(seed)
    held = [-(-n // page) for n in kv_lens]
    pages = sum(held) + 2
    order = rng.permutation(pages)
    table = np.full((len(kv_lens), cols or max(max(held, default=0), 1)), -1, dtype=np.int32)
    pool = rng.integers(0, 256, (pages, heads_k, page // 16 * 20 * dim)).astype(np.uint8)  # unused tokens: anything
    at, keys, values = 0, [], []
    for b, n in enumerate(kv_lens):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
        k = rng.standard_normal((n, heads_k, dim)).astype(np.float16)
        v = (rng.standard_normal((n, heads_k, dim)) * v_scale).astype(np.float16)
        k[:, :, 7] *= 10
        pos = np.arange(n)
        slots = table[b, pos // page].astype(np.int64) * page + pos % page
        ora.append(pool, k, v, slots)
        k, v = ora.read(pool, slots, dim)
        keys.append(k)
        values.append(v)
    to = lambda x: torch.from_numpy(x).to(dev)  # noqa: E731
    return to(pool), to(table), torch.tensor(kv_lens, dtype=torch.int32, device=dev), keys, values


def _queries(dev, new, heads, dim, seed, pad=0):
    q = torch.randn((sum(new) + pad, heads, dim), generator=torch.Generator().manual_seed(seed)).half().to(dev)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=dev)
    return q, cu


def _assert_close(out, q, cu, keys, values, scale, causal=True, mask=None):
    out, q, cu = out.double().cpu().numpy(), q.cpu().numpy(), cu.cpu().numpy()
    for b in range(len(keys)):
        rows = slice(cu[b], cu[b + 1])
        ref, bound = ora.attention(q[rows], keys[b], values[b], len(keys[b]), scale, causal,
                                   None if mask is None else mask[b].cpu().numpy())
        err = np.abs(out[rows] - ref)
        assert (err <= bound).all(), (b, float((err / bound).max()), float(err.max()))


@pytest.mark.parametrize("kv_lens,new,heads,heads_k,dim,page", [
    ([1], [1], 1, 1, 64, 16),
    ([16, 17, 15, 32, 33], [1] * 5, 8, 1, 128, 16),
    ([300, 1, 77], [1] * 3, 28, 4, 128, 32),
    ([513], [1], 24, 8, 128, 64),
    ([127, 128, 129], [1] * 3, 6, 2, 64, 48),
    ([40, 500, 3], [15, 7, 3], 8, 2, 64, 32),
    ([260, 31], [5, 31], 14, 2, 128, 128),
    ([200, 50], [3, 2], 18, 1, 64, 16),
    ([20, 90], [40, 33], 4, 4, 128, 256),
    ([3000, 100], [1, 1], 4, 2, 128, 64),
])
def test_attention_matches_the_oracle(cuda_device, kv_lens, new, heads, heads_k, dim, page):
    from tilemix_b200.attention.kv4 import kv4_attention

    pool, table, lens, keys, values = _cache(cuda_device, kv_lens, heads_k, dim, page, seed=sum(kv_lens))
    q, cu = _queries(cuda_device, new, heads, dim, seed=1)
    out = kv4_attention(q, pool, table, lens, cu, max(new))
    _assert_close(out, q, cu, keys, values, dim ** -0.5)
    if max(new) == 1:
        assert torch.equal(kv4_attention(q, pool, table, lens), out)


def test_attention_options(cuda_device):
    """All keys visible, another scale, strided q and out, wide tables and bounds: the split changes, the result does not
    beyond rounding."""
    from tilemix_b200.attention.kv4 import kv4_attention

    pool, table, lens, keys, values = _cache(cuda_device, [700, 60], 2, 128, 32, seed=9, cols=2000)
    q, cu = _queries(cuda_device, [4, 9], 6, 128, seed=2)
    wide = torch.cat([q, q], 2)[..., 128:]
    store = torch.full((13, 8, 128), 7.0, dtype=torch.float16, device=cuda_device)
    got = kv4_attention(wide, pool, table, lens, cu, 9, causal=False, sm_scale=0.3, out=store[:, 1:7])
    assert got.data_ptr() == store[:, 1:7].data_ptr()
    _assert_close(got, q, cu, keys, values, 0.3, causal=False)
    assert (store[:, 0] == 7).all() and (store[:, 7] == 7).all()
    _assert_close(kv4_attention(q, pool, table, lens, cu, 9, max_kv_len=700), q, cu, keys, values, 128 ** -0.5)


def test_many_splits(cuda_device):
    """One long request: the key axis is cut, the parts are joined."""
    from tilemix_b200.attention.kv4 import kv4_attention

    pool, table, lens, keys, values = _cache(cuda_device, [9000], 1, 64, 64, seed=4)
    q, cu = _queries(cuda_device, [2], 5, 64, seed=3)
    q *= 3  # a sharper softmax: parts of very different weight
    _assert_close(kv4_attention(q, pool, table, lens, cu, 2), q, cu, keys, values, 64 ** -0.5)


@pytest.mark.parametrize("dim", [64, 128])
def test_masked_keys_and_empty_rows(cuda_device, dim):
    """Masked keys may hold NaN or infinities; rows without a key are 0; a key behind the mask's columns is excluded."""
    from tilemix_b200.attention.kv4 import kv4_append, kv4_attention

    kv_lens, new = [100, 600, 40, 0, 5], [1, 6, 3, 2, 9]
    pool, table, lens, keys, values = _cache(cuda_device, kv_lens, 2, dim, 16, seed=6)
    mask = torch.rand((5, 580), generator=torch.Generator().manual_seed(2)) > 0.4
    mask[0, :99] = False
    mask[2] = False
    mask = mask.to(cuda_device)
    mask[1, 50:60] = False
    bad = torch.full((10, 2, dim), float("nan"), dtype=torch.float16, device=cuda_device)
    bad[:, :, ::2] = float("inf")
    slots = table[1, torch.arange(50, 60) // 16].long() * 16 + torch.arange(50, 60, device=cuda_device) % 16
    kv4_append(bad, bad, pool, slots)
    q, cu = _queries(cuda_device, new, 8, dim, seed=5, pad=2)
    out = torch.full_like(q, 3.0)
    kv4_attention(q, pool, table, lens, cu, 9, key_mask=mask, out=out)
    _assert_close(out, q, cu, keys, values, dim ** -0.5, mask=mask)
    assert (out[7:10] == 0).all() and (out[10:12] == 0).all() and (out[12:16] == 0).all()
    assert (out[-2:] == 3).all()  # rows behind the last request


@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_finite_stays_with_the_rows_that_see_it(cuda_device, dim):
    """New tokens whose keys or values are infinite or NaN leave the rows in front of them alone (their weight there is 0,
    and 0 times NaN is NaN); the rows that see them are NaN, a value's in its group of channels only."""
    from tilemix_b200.attention.kv4 import kv4_append, kv4_attention

    kv_lens, new = [70, 33, 9, 40], [6, 33, 4, 20]
    pool, table, lens, keys, values = _cache(cuda_device, kv_lens, 2, dim, 16, seed=9)

    def spoil(b, pos, k_too):
        x = torch.from_numpy(np.stack([keys[b][pos], values[b][pos]])).half().to(cuda_device)[:, None]
        x[1, :, 0, 40] = float("inf")
        values[b][pos, 0, 32:64] = np.nan
        if k_too:
            x[0, :, 1, 3] = float("nan")
            keys[b][pos, 1, :32] = np.nan
        kv4_append(x[0], x[1], pool, table[b, pos // 16:pos // 16 + 1].long() * 16 + pos % 16)

    spoil(0, 67, False)
    spoil(1, 32, True)
    spoil(1, 7, False)
    spoil(2, 8, True)
    spoil(3, 25, True)
    q, cu = _queries(cuda_device, new, 8, dim, seed=6)
    out = kv4_attention(q, pool, table, lens, cu, 33)
    ends = cu.tolist()
    for b, n in enumerate(new):
        rows = slice(ends[b], ends[b + 1])
        with np.errstate(invalid="ignore"):
            ref, bound = ora.attention(q[rows].cpu().numpy(), keys[b], values[b], kv_lens[b], dim ** -0.5, True)
        got = out[rows].double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(ref)), b
        fine = ~np.isnan(ref)
        assert np.isnan(ref).any() and fine[0].all() == (b in (0, 1, 2, 3))
        assert (np.abs(got - ref)[fine] <= bound[fine]).all(), b


@pytest.mark.parametrize("v_scale", [1e-5, 300.0])
def test_small_and_large_values(cuda_device, v_scale):
    from tilemix_b200.attention.kv4 import kv4_attention

    pool, table, lens, keys, values = _cache(cuda_device, [400], 1, 128, 32, seed=8, v_scale=v_scale)
    q, cu = _queries(cuda_device, [1], 4, 128, seed=7)
    _assert_close(kv4_attention(q, pool, table, lens), q, cu, keys, values, 128 ** -0.5)


def test_pages_outside_the_pool_are_left_out(cuda_device):
    """A page number outside the pool: its keys do not count, the error word says 12, nothing is read there."""
    from tilemix_b200.attention.kv4 import kv4_attention

    pool, table, lens, keys, values = _cache(cuda_device, [100], 2, 64, 16, seed=10)
    q, cu = _queries(cuda_device, [1], 4, 64, seed=8)
    for page in (-1, pool.shape[0], 2**31 - 1):
        broken = table.clone()
        broken[0, 2] = page
        out = kv4_attention(q, pool, broken, lens)
        assert _error_code() == 12
        left = torch.ones((1, 100), dtype=torch.bool)
        left[0, 32:48] = False
        _assert_close(out, q, cu, keys, values, 64 ** -0.5, mask=left)


def test_lengths_beyond_the_table_are_reported(cuda_device):
    from tilemix_b200.attention.kv4 import kv4_attention

    pool, table, lens, keys, values = _cache(cuda_device, [64], 1, 64, 16, seed=11)
    q, cu = _queries(cuda_device, [1], 2, 64, seed=9)
    out = kv4_attention(q, pool, table, lens + 1000, causal=False)
    assert _error_code() == 11
    _assert_close(out, q, cu, keys, values, 64 ** -0.5, causal=False)


def test_more_query_tokens_than_said_are_reported(cuda_device):
    from tilemix_b200.attention.kv4 import kv4_attention

    pool, table, lens, keys, values = _cache(cuda_device, [64, 70], 1, 64, 16, seed=13)
    q, cu = _queries(cuda_device, [3, 5], 2, 64, seed=11)
    out = torch.full_like(q, 3.0)
    kv4_attention(q, pool, table, lens, cu, 4, out=out)
    assert _error_code() == 11 and (out[-1] == 3).all() and not (out[:-1] == 3).all(-1).any()


def test_no_rows_and_no_requests(cuda_device):
    from tilemix_b200.attention.kv4 import kv4_append, kv4_attention, kv4_pool, kv4_read

    pool = kv4_pool(1, 16, 2, 64, cuda_device)
    none = torch.zeros(0, dtype=torch.int64, device=cuda_device)
    k = torch.zeros((0, 2, 64), dtype=torch.float16, device=cuda_device)
    kv4_append(k, k, pool, none)
    assert kv4_read(pool, none, 64)[0].shape == (0, 2, 64)
    empty = torch.zeros((0, 1), dtype=torch.int32, device=cuda_device)
    out = kv4_attention(torch.zeros((0, 4, 64), dtype=torch.float16, device=cuda_device), pool, empty, empty[:, 0])
    assert out.shape == (0, 4, 64)


def test_a_step_in_a_graph_grows_the_cache(cuda_device):
    """Tables, append and attention of a decode step captured once and replayed: each replay adds a token, equal to the
    eager steps bit for bit; a second graph on its own stream shares nothing with the first."""
    from tilemix_b200.attention.kv4 import build_block_tables, kv4_append, kv4_attention, kv4_pool

    dev, page, heads_k, dim, batch, steps = cuda_device, 16, 2, 64, 3, 20
    gen = torch.Generator().manual_seed(0)
    feed = [torch.randn((3, batch, heads_k, dim), generator=gen).half().to(dev) for _ in range(steps)]

    class Server:
        def __init__(self):
            self.pool = kv4_pool(12, page, heads_k, dim, dev)
            self.ring = torch.arange(12, dtype=torch.int32, device=dev)
            self.span = torch.tensor([0, 12], device=dev)
            self.table = torch.full((batch, 4), -1, dtype=torch.int32, device=dev)
            self.lens = torch.zeros(batch, dtype=torch.int32, device=dev)
            self.one = torch.ones(batch, dtype=torch.int32, device=dev)
            self.x = torch.zeros((3, batch, heads_k, dim), dtype=torch.float16, device=dev)

        def step(self):
            t = build_block_tables(self.lens, self.one, self.table, self.ring, self.span, page_size=page,
                                   max_new_tokens=batch)
            kv4_append(self.x[1], self.x[2], self.pool, t.slots)
            out = kv4_attention(self.x[0], self.pool, self.table, t.kv_lens)
            self.lens.copy_(t.kv_lens)
            self.span.copy_(t.free_span)
            return out

        def reset(self):
            self.span.copy_(torch.tensor([0, 12]))
            self.table.fill_(-1)
            self.lens.zero_()

    eager = Server()
    want = []
    for x in feed:
        eager.x.copy_(x)
        want.append(eager.step().clone())
    servers, graphs, outs = [Server(), Server()], [], []
    for s in servers:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            s.step()
        side.synchronize()
        s.reset()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(s.step())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in servers]
    torch.cuda.synchronize()
    for i, x in enumerate(feed):
        for s, graph, st in zip(servers, graphs, streams):
            with torch.cuda.stream(st):
                s.x.copy_(x)
                graph.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, want[i])


def test_repeated_calls_are_identical(cuda_device):
    from tilemix_b200.attention.kv4 import kv4_attention

    pool, table, lens, _, _ = _cache(cuda_device, [2000, 700], 2, 64, 32, seed=12)
    q, cu = _queries(cuda_device, [2, 5], 6, 64, seed=10)
    first = kv4_attention(q, pool, table, lens, cu, 5)
    for _ in range(5):
        assert torch.equal(kv4_attention(q, pool, table, lens, cu, 5), first)


# ---------------------------------------------------------------------------------------------- bounds that do not hold
def _near(got, ref, bound):
    """Whether every element is within its bound (a NaN is not)."""
    return bool((np.abs(got - ref) <= bound).all())


@pytest.mark.parametrize("dim", [64, 128])
def test_queries_beyond_their_bound_do_not_shift_the_others(cuda_device, dim):
    """The rows of a request that has more than max_seqlen_q see the keys that they see without the bound."""
    from tilemix_b200.attention.kv4 import kv4_attention

    kv_lens, new, most = [64, 300, 70, 9], [3, 20, 5, 6], 4
    pool, table, lens, keys, values = _cache(cuda_device, kv_lens, 2, dim, 16, seed=21)
    q, cu = _queries(cuda_device, new, 4, dim, seed=21)
    out = torch.full_like(q, 3.0)
    kv4_attention(q, pool, table, lens, cu, most, out=out)
    assert _error_code() == 11
    got, rows = out.double().cpu().numpy(), q.cpu().numpy()
    ends = cu.tolist()
    for b, n in enumerate(new):
        ref, bound = ora.attention(rows[ends[b]:ends[b + 1]], keys[b], values[b], kv_lens[b], dim ** -0.5, True)
        served = min(n, most)
        assert _near(got[ends[b]:ends[b] + served], ref[:served], bound[:served]), b
        assert (got[ends[b] + served:ends[b + 1]] == 3).all(), b


@pytest.mark.parametrize("more", [1, 3, 1000])
def test_keys_beyond_their_bound_do_not_shift_the_others(cuda_device, more):
    """A request of more keys than max_kv_len (or the table) holds: a row sees the keys up to its own place that are there."""
    from tilemix_b200.attention.kv4 import kv4_attention

    kv_lens, new = [64, 33], [5, 7]
    pool, table, lens, keys, values = _cache(cuda_device, kv_lens, 2, 64, 16, seed=22, cols=4)
    q, cu = _queries(cuda_device, new, 4, 64, seed=22)
    longer = lens.clone()
    longer[0] += more
    out = kv4_attention(q, pool, table, longer, cu, 7, max_kv_len=64)
    assert _error_code() == 11
    got, rows = out.double().cpu().numpy(), q.cpu().numpy()
    for i in range(5):  # row i sees min(64 + more - 5 + i + 1, 64) keys
        seen = min(64, 64 + more - 5 + i + 1)
        ref, bound = ora.attention(rows[i:i + 1], keys[0][:seen], values[0][:seen], seen, 64 ** -0.5, True)
        assert _near(got[i:i + 1], ref, bound), i
    ref, bound = ora.attention(rows[5:], keys[1], values[1], 33, 64 ** -0.5, True)
    assert _near(got[5:], ref, bound)


@pytest.mark.parametrize("offsets,served", [
    ([0, 3, 2, 2], [0, 2]),   # the second request's end is in front of its start
    ([0, 3, 5, 9], [0, 1]),   # the third one's rows run past q
    ([-1, 1, 3, 5], [1, 2]),  # the first one's begin in front of q
    ([0, -2**31, -5, -5], []), ([2**31 - 1, -2**31, 7, 7], []),
    ([0, 2, 4, 6], [0, 1, 2]),
])
def test_offsets_that_do_not_hold_are_reported(cuda_device, offsets, served):
    """A request whose rows are not all rows of q is left out, and the error word says so."""
    from tilemix_b200.attention.kv4 import kv4_attention

    pool, table, lens, keys, values = _cache(cuda_device, [40, 50, 60], 2, 64, 16, seed=23)
    q, _ = _queries(cuda_device, [6], 4, 64, seed=23)
    out = torch.full_like(q, 3.0)
    kv4_attention(q, pool, table, lens, torch.tensor(offsets, dtype=torch.int32, device=cuda_device), 4, out=out)
    assert _error_code() == (0 if offsets[0] == 0 and offsets[3] == 6 else 11)
    got, rows = out.double().cpu().numpy(), q.cpu().numpy()
    free = np.ones(6, dtype=bool)
    for b in served:
        at = slice(offsets[b], offsets[b + 1])
        free[at] = False
        ref, bound = ora.attention(rows[at], keys[b], values[b], len(keys[b]), 64 ** -0.5, True)
        assert _near(got[at], ref, bound), b
    assert (got[free] == 3).all()


def test_negative_lengths_are_reported(cuda_device):
    """A negative length counts as no key: rows of 0, and the error word says 11."""
    from tilemix_b200.attention.kv4 import kv4_attention

    pool, table, lens, keys, values = _cache(cuda_device, [40, 50], 2, 64, 16, seed=24)
    q, cu = _queries(cuda_device, [2, 3], 4, 64, seed=24)
    for wrong in (-1, -2**31):
        broken = lens.clone()
        broken[0] = wrong
        for causal in (True, False):
            out = kv4_attention(q, pool, table, broken, cu, 3, causal=causal)
            assert _error_code() == 11 and (out[:2] == 0).all()
            ref, bound = ora.attention(q[2:].cpu().numpy(), keys[1], values[1], 50, 64 ** -0.5, causal)
            assert _near(out[2:].double().cpu().numpy(), ref, bound)


@pytest.mark.parametrize("heads,dim", [(1, 64), (2, 128)])
def test_strides_that_are_not_used_may_be_any(cuda_device, heads, dim):
    """One token, or one head: its row starts on 16 bytes whatever the stride to the next one would be."""
    from tilemix_b200.attention.kv4 import kv4_append, kv4_attention, kv4_pool, kv4_read

    g = torch.Generator().manual_seed(4)
    wide = torch.randn((2, 3 * heads * dim + 4), generator=g).half().to(cuda_device)
    one = wide.as_strided((1, heads, dim), (3 * heads * dim + 4, dim, 1))
    pool, table = kv4_pool(2, 16, heads, dim, cuda_device), torch.zeros((1, 1), dtype=torch.int32, device=cuda_device)
    kv4_append(one, one, pool, torch.tensor([0], device=cuda_device))
    k, v = kv4_read(pool, torch.tensor([0], device=cuda_device), dim)
    ref = np.zeros(pool.shape, dtype=np.uint8)
    ora.append(ref, one.cpu().numpy(), one.cpu().numpy(), [0])
    assert np.array_equal(pool.cpu().numpy(), ref)
    out = torch.empty_like(wide).as_strided((1, heads, dim), (3 * heads * dim + 4, dim, 1))
    kv4_attention(one, pool, table, torch.tensor([1], dtype=torch.int32, device=cuda_device), out=out)
    assert torch.equal(out, v)  # a single key: its value
    rows = torch.randn((5, dim), generator=g).half().to(cuda_device)
    single = rows.as_strided((5, 1, dim), (dim, 3, 1))
    pool = kv4_pool(1, 16, 1, dim, cuda_device)
    kv4_append(single, single, pool, torch.arange(5, device=cuda_device))
    k, v = kv4_read(pool, torch.arange(5, device=cuda_device), dim)
    ref = np.zeros(pool.shape, dtype=np.uint8)
    ora.append(ref, rows[:, None].cpu().numpy(), rows[:, None].cpu().numpy(), range(5))
    assert np.array_equal(pool.cpu().numpy(), ref)
    out = kv4_attention(single, pool, table.expand(5, 1), torch.ones(5, dtype=torch.int32, device=cuda_device))
    assert torch.equal(out, v[:1].expand(5, 1, dim))


def test_errors_of_another_stream_are_read(cuda_device):
    """device_error_code waits for the device, not for the current stream alone."""
    from tilemix_b200.attention.kv4 import kv4_append, kv4_pool

    x = torch.ones((1, 1, 64), dtype=torch.float16, device=cuda_device)
    pool, slot = kv4_pool(1, 16, 1, 64, cuda_device), torch.tensor([99], device=cuda_device)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1000)
        kv4_append(x, x, pool, slot - 99)  # the kernels are loaded, which waits for the device
        torch.cuda.synchronize()
        torch.cuda._sleep(50_000_000)  # some 25 ms
        kv4_append(x, x, pool, slot)
    assert _error_code() == 13
    with torch.cuda.stream(side):
        assert _error_code() == 0  # cleared for every stream
