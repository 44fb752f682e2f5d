"""GPU tests of the 4-bit cache at sizes where a CTA of the attention has many chunks, several runs and rings that wrap,
where the requests outnumber a warp's lanes, and where the block tables of a long prefill are filled by many CTAs.
The cached values are decoded from the pool's bytes in 64 bits, by the offsets of the oracle's layout."""
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


# ---------------------------------------------------------------------------------------------- attention
def _filled_cache(dev, kv_lens, heads, dim, page, seed):
    """A pool of random bytes with the requests' normal values (outliers in one channel) on pages in any order."""
    from tilemix_b200.attention.kv4 import kv4_append

    g = torch.Generator(device=dev).manual_seed(seed)
    held = [-(-n // page) for n in kv_lens]
    pages = sum(held) + 2
    order = torch.randperm(pages, generator=g, device=dev).int()
    table = torch.full((len(kv_lens), max(held) + 1), -1, dtype=torch.int32, device=dev)
    pool = torch.randint(0, 256, (pages, heads, page // 16 * 20 * dim), generator=g, device=dev, dtype=torch.uint8)
    at = 0
    for b, n in enumerate(kv_lens):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
        k, v = (torch.randn((n, heads, dim), generator=g, device=dev).half() for _ in range(2))
        k[:, :, 7] *= 10
        kv4_append(k, v, pool, _slots(table[b], torch.arange(n, device=dev), page))
    return pool, table, torch.tensor(kv_lens, dtype=torch.int32, device=dev)


def _slots(row, pos, page):
    return row[pos // page].long() * page + pos % page


def _decoded(pool, row, pos, dim):
    """The values at positions ``pos`` of a request, 64 bits [positions, heads, dim] each."""
    dev, heads, page = pool.device, pool.shape[1], pool.shape[2] // (20 * dim) * 16
    offsets = [torch.from_numpy(np.stack(x)).to(dev) for x in zip(*(ora.block_offsets(dim, t) for t in range(16)))]
    blocks = pool.view(pool.shape[0], heads, page // 16, 20 * dim)[row[pos // page].long(), :, pos % page // 16]
    tok, shift = pos % 16, (torch.arange(dim, device=dev) % 2 * 4).to(torch.uint8)
    take = lambda at: blocks.gather(2, at[tok][:, None].expand(-1, heads, -1))  # noqa: E731

    def half(at):
        return (take(at).int() | take(at + 1).int() << 8).to(torch.int16).view(torch.float16).double()

    def values(codes, scale, low):
        n = (take(offsets[codes]) >> shift & 15).double().unflatten(2, (-1, 32))
        return (n * half(offsets[scale])[..., None] + half(offsets[scale] + low)[..., None]).flatten(2)

    return values(0, 2, 2), values(1, 3, 8)


def _reference(q, k, v, sees, scale, steps):
    """64-bit attention of rows q [n, heads_q, dim] over k / v [keys, heads, dim], row i over those with sees[i], and
    the oracle's bound on what fp16 operands change (ora.attention), with the sums of a long run: a warp has at most
    ``steps`` steps, in each of which a lane adds four weights to its sum (2^-24 of it each) and the tensor core two
    products of 16 keys (2^-22 of the sum's magnitude each, were its additions cut off), and both are rescaled (2^-24):
    under 4 * 2^-22 a step, and 64 * 2^-22 for the exponentials, the merge of the warps and the join."""
    n, heads_q, dim = q.shape
    heads = k.shape[1]
    q = q.double().view(n, heads, -1, dim)
    s = torch.einsum("nhgd,khd->nhgk", q, k) * scale
    groups = k.unflatten(2, (-1, 32))
    spread = (groups.amax(-1) - groups.amin(-1)) / 15
    d = torch.einsum("nhgj,khj->nhgk", q.abs().unflatten(3, (-1, 32)).sum(-1), spread) * 2.0 ** -10
    d = (d + 2.0 ** -21 * torch.einsum("nhgd,khd->nhgk", q.abs(), k.abs())) * scale
    sees = sees[:, None, None]
    s, d = torch.where(sees, s, -torch.inf), torch.where(sees, d, 0.0).amax(-1)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -torch.inf, top, 0.0))
    total = p.sum(-1)[..., None].clamp(min=1e-300)
    out, near = torch.einsum("nhgk,khd->nhgd", p, v) / total, torch.einsum("nhgk,khd->nhgd", p, v.abs()) / total
    every = torch.einsum("nhgk,khd->nhgd", (p > 0).double(), v.abs()) / total
    sums = 2.0 ** -22 * (4 * steps + 64)
    bound = near * (torch.expm1(2 * d)[..., None] + 3 * 2.0 ** -11 + sums) + 2.0 ** -25 * every
    bound += 2.0 ** -11 * out.abs() + 2.0 ** -25
    return out.reshape(n, heads_q, dim), bound.reshape(n, heads_q, dim)


def _check_attention(dev, kv_lens, new, heads_q, heads, dim, page, seed, masked=False, absent=(), spoiled=()):
    """``absent``: (request, table column)s whose page number is none; ``spoiled``: requests whose masked keys are not
    finite."""
    from tilemix_b200.attention.kv4 import kv4_append, kv4_attention

    pool, table, lens = _filled_cache(dev, kv_lens, heads, dim, page, seed)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    q = torch.randn((sum(new) + 3, heads_q, dim), generator=g, device=dev).half()
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=dev)
    mask = None
    if masked:
        mask = torch.rand((len(kv_lens), max(kv_lens)), generator=g, device=dev) > 0.1
        start = (torch.rand(len(kv_lens), 1, generator=g, device=dev) * 0.6 * lens[:, None]).long()
        mask &= torch.arange(mask.shape[1], device=dev)[None] >= start
    for b in spoiled:
        pos = (~mask[b, :kv_lens[b]]).nonzero()[:, 0]
        bad = torch.full((len(pos), heads, dim), float("nan"), dtype=torch.float16, device=dev)
        bad[:, :, ::2] = float("inf")
        kv4_append(bad, bad, pool, _slots(table[b], pos, page))
    broken = table.clone()
    for b, col in absent:
        broken[b, col] = -1
    out = torch.full_like(q, 3.0)

    def call():
        kv4_attention(q, pool, broken, lens, cu, max(new), key_mask=mask, max_kv_len=max(kv_lens), out=out)

    call()
    assert _error_code() == (12 if absent else 0)
    assert (out[sum(new):] == 3).all()
    first, ends = out.clone(), cu.tolist()
    for b, (length, n) in enumerate(zip(kv_lens, new)):
        if n == 0:
            continue
        pos = torch.arange(length, device=dev)
        keep = torch.ones(length, dtype=torch.bool, device=dev) if mask is None else mask[b, :length].clone()
        for at, col in absent:
            if at == b:
                keep[col * page:(col + 1) * page] = False
        pos = pos[keep]
        rows = slice(ends[b], ends[b + 1])
        if len(pos) == 0:
            assert (out[rows] == 0).all(), b
            continue
        k, v = _decoded(pool, table[b], pos, dim)
        sees = pos[None] < length - n + 1 + torch.arange(n, device=dev)[:, None]
        ref, bound = _reference(q[rows], k, v, sees, dim ** -0.5, -(-length // 128))
        err = out[rows].double() - ref
        assert bool((err.abs() <= bound).all()), (b, length, n, float((err.abs() / bound).max()))
        # Over a request's outputs the roundings of v, p and the result are independent: each at most 2^-11 of its
        # term, evenly spread, so 2^-11 / sqrt(3) in the mean square, and together 2^-11. Twice that is allowed. A key
        # too many or too few among n changes the outputs by about 1 / sqrt(n) of their size.
        assert float(err.norm()) <= 2.0 ** -10 * float(ref.norm()), (b, length, n, float(err.norm() / ref.norm()))
    for _ in range(3):
        out.fill_(3.0)
        call()
        assert torch.equal(out, first)
    _error_code()


def _mixed(seed, batch, low, high, new, empty=0.1):
    """Lengths of a server's requests, some without a key and some without a query token."""
    rng = np.random.default_rng(seed)
    kv = rng.integers(low, high + 1, batch)
    kv[rng.random(batch) < empty] = 0
    n = rng.integers(1, new + 1, batch)
    n[rng.random(batch) < empty] = 0
    return kv.tolist(), n.tolist()


@pytest.mark.parametrize("batch,low,high,new,heads_q,heads,dim,page", [
    (90, 1, 6000, 1, 24, 8, 128, 64),   # some 40 chunks a CTA, of several requests
    (64, 2900, 3100, 1, 8, 8, 64, 16),  # one row a KV head
    (300, 1, 700, 2, 8, 2, 64, 48),     # ten requests a lane of the scan
    (36, 100, 9000, 4, 12, 2, 128, 128),
])
def test_attention_of_a_full_server(cuda_device, batch, low, high, new, heads_q, heads, dim, page):
    kv, n = _mixed(batch, batch, low, high, new)
    _check_attention(cuda_device, kv, n, heads_q, heads, dim, page, seed=batch)


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_several_tokens_with_masked_keys(cuda_device, dim):
    kv, n = _mixed(7, 40, 500, 9000, 15)
    kv[3], n[3], kv[11], n[11] = 6000, 4, 7777, 15
    _check_attention(cuda_device, kv, n, 16, 4, dim, 32, seed=7, masked=True, spoiled=(3, 11))


@pytest.mark.parametrize("kv_lens,new,heads_q,heads,dim,page", [
    ([70000, 66001], [15, 9], 32, 16, 64, 64),  # over 64 steps a warp and run: page addresses looked up three times
    ([131072, 50], [1, 1], 32, 8, 128, 64),     # one request on every CTA
    ([40000, 0, 39990], [1, 2, 1], 3, 1, 64, 16),
])
def test_attention_of_long_requests(cuda_device, kv_lens, new, heads_q, heads, dim, page):
    _check_attention(cuda_device, kv_lens, new, heads_q, heads, dim, page, seed=len(kv_lens))


def test_pages_missing_far_behind_are_left_out(cuda_device):
    _check_attention(cuda_device, [70000, 66001], [3, 2], 32, 16, 64, 16, seed=3,
                     absent=((0, 0), (0, 4000), (0, 4001), (0, 4374), (1, 2111), (1, 4125)))


def test_attention_of_many_tokens_over_a_filled_cache(cuda_device):
    """A second turn: hundreds of new tokens behind thousands of cached ones."""
    _check_attention(cuda_device, [5000, 3333, 700], [300, 1, 512], 6, 2, 64, 64, seed=9)
    _check_attention(cuda_device, [2100, 1300], [65, 129], 8, 2, 128, 32, seed=10, masked=True)


@pytest.mark.parametrize("bits", [10.0, 16.3, 20.3, 24.6, 25.5, 30.0])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_small_weights_behind_a_large_one(cuda_device, dim, bits):
    """A first key that draws nearly all of a row's attention, and 8192 others with 2^-bits of its weight each, whose
    values are what the row sees: p = 2^-bits has to reach the product with v. Keys and values are constant in a row, so
    the cache holds them exactly. Weights are held in fp16 times 2^15: to 2^-11 of them, and to 2^-40 of the largest;
    v = 1 is exact, the result is rounded once, and a score of under 32 is off by 2^-17 at most in fp32."""
    from tilemix_b200.attention.kv4 import kv4_append, kv4_attention, kv4_pool

    n, page, batch, heads = 8193, 64, 60, 8
    pages = -(-n // page)
    pool = kv4_pool(pages, page, heads, dim, cuda_device)
    table = torch.arange(pages, device=cuda_device).int().expand(batch, pages)
    k = torch.zeros((n, heads, dim), dtype=torch.float16, device=cuda_device)
    v = torch.ones_like(k)
    k[0] = bits * np.log(2) / dim ** 0.5
    v[0] = 0
    kv4_append(k, v, pool, torch.arange(n, device=cuda_device))
    q = torch.ones((batch, 3 * heads, dim), dtype=torch.float16, device=cuda_device)
    out = kv4_attention(q, pool, table, torch.full((batch,), n, dtype=torch.int32, device=cuda_device))
    rest = (n - 1) * np.exp(-float(k[0, 0, 0]) * dim ** 0.5)
    want = rest / (1 + rest)
    bound = want * (2 * 2.0 ** -11 + 2.0 ** -16) + (n - 1) * 2.0 ** -40 + 2.0 ** -25
    assert float((out.double() - want).abs().max()) <= bound, (want, out.min().item(), out.max().item())


@pytest.mark.parametrize("heads,dim,page", [(8, 128, 64), (3, 64, 48)])
def test_a_pool_beyond_32_bits(cuda_device, heads, dim, page):
    """Slots whose bytes lie more than 2^32 into the pool, and in front of that."""
    from tilemix_b200.attention.kv4 import kv4_append, kv4_attention, kv4_read

    row = page // 16 * 20 * dim
    pages = (2**32 + 2**29) // (heads * row)
    pool = torch.empty((pages, heads, row), dtype=torch.uint8, device=cuda_device)
    edge = 2**32 // (heads * row)  # the page that holds byte 2^32
    table = torch.tensor([[pages - 1, 0, edge, edge + 1], [edge - 1, pages - 2, 2**31 // (heads * row), 7]],
                         dtype=torch.int32, device=cuda_device)
    n = 4 * page - 5
    g = torch.Generator(device=cuda_device).manual_seed(1)
    slots = torch.cat([_slots(table[b], torch.arange(n, device=cuda_device), page) for b in range(2)])
    k, v = (torch.randn((2 * n, heads, dim), generator=g, device=cuda_device).half() for _ in range(2))
    kv4_append(k, v, pool, slots)
    got = kv4_read(pool, slots, dim)
    small = torch.empty((8, heads, row), dtype=torch.uint8, device=cuda_device)
    few = torch.arange(8, dtype=torch.int32, device=cuda_device).view(2, 4)
    near = torch.cat([_slots(few[b], torch.arange(n, device=cuda_device), page) for b in range(2)])
    kv4_append(k, v, small, near)
    assert all(torch.equal(a, b) for a, b in zip(got, kv4_read(small, near, dim)))
    q = torch.randn((2, heads * 2, dim), generator=g, device=cuda_device).half()
    lens = torch.full((2,), n, dtype=torch.int32, device=cuda_device)
    assert torch.equal(kv4_attention(q, pool, table, lens), kv4_attention(q, small, few, lens))


# ---------------------------------------------------------------------------------------------- block tables
def _tables_case(cached, new, page, seed, extra_pages=5):
    rng = np.random.default_rng(seed)
    cached, new = np.asarray(cached), np.asarray(new)
    held, total = -(-cached // page), -(-(cached + new) // page)
    capacity = int(total.sum()) + extra_pages
    order = rng.permutation(capacity).astype(np.int32)
    table = np.full((len(cached), int(total.max()) + 2), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    head, free = int(rng.integers(0, capacity)), order[at:]
    ring = np.full(capacity, -7, dtype=np.int32)
    ring[(head + np.arange(len(free))) % capacity] = free
    return cached, new, table, ring, np.array([head, head + len(free)], dtype=np.int64)


def _build(dev, cached, new, table, ring, span, page, rows):
    from tilemix_b200.attention.kv4 import build_block_tables

    to = lambda x, t: torch.tensor(np.asarray(x), dtype=t, device=dev)  # noqa: E731
    tab = to(table, torch.int32)
    got = build_block_tables(to(cached, torch.int32), to(new, torch.int32), tab, to(ring, torch.int32),
                             to(span, torch.int64), page_size=page, max_new_tokens=rows)
    return [x.cpu().numpy() for x in got] + [tab.cpu().numpy()]


def _ragged(seed, batch, cached, new):
    rng = np.random.default_rng(seed)
    n = rng.integers(1, new, batch)
    n[rng.random(batch) < 0.2] = 0
    return rng.integers(0, cached, batch), n


@pytest.mark.parametrize("seed,batch,cached,new,page,more", [
    (1, 60, 300, 4000, 48, 5),      # some 90,000 tokens: four a thread
    (2, 1500, 90, 130, 16, 0),      # pages and requests that end inside a thread's four
    (3, 5, 5000, 400000, 64, 3),    # more than the grid has threads for: several rounds
    (4, 3, 10, 20, 16, 76001),      # rows behind the last request, an odd number of them
    (5, 8192, 20, 200, 32, 2),
])
def test_tables_of_long_prefills(cuda_device, seed, batch, cached, new, page, more):
    case = _tables_case(*_ragged(seed, batch, cached, new), page, seed)
    rows = int(case[1].sum()) + more
    assert rows > 148 * 512
    got, ref = _build(cuda_device, *case, page, rows), ora.build_block_tables(*case, page, rows)
    for g, r in zip(got, ref[:6]):
        assert np.array_equal(g, r)


@pytest.mark.parametrize("why", ["pages", "columns", "slots", "negative"])
def test_tables_of_long_prefills_are_all_or_nothing(cuda_device, why):
    cached, new, table, ring, span = _tables_case(*_ragged(6, 60, 300, 4000), 48, 6, extra_pages=0)
    rows = int(new.sum()) + 2
    if why == "pages":
        span[1] -= 1
    elif why == "columns":
        table = table[:, :-3]
    elif why == "slots":
        rows -= 3
    else:
        cached[7] = -1
    got = _build(cuda_device, cached, new, table, ring, span, 48, rows)
    assert _error_code() == 11
    assert (got[0] == -1).all() and (got[1] == 0).all() and (got[2] == 0).all()
    assert np.array_equal(got[3], cached) and np.array_equal(got[4], span) and np.array_equal(got[5], table)


def test_tables_into_memory_that_is_not_on_16_bytes(cuda_device):
    """As the C ABI allows it; nothing is written beside the outputs."""
    from tilemix_b200._lib import TmBlockTablesParams, launcher, packer

    page, case = 32, _tables_case(*_ragged(8, 50, 100, 5000), 32, 8)
    rows = int(case[1].sum()) + 3
    assert rows > 148 * 512
    to = lambda x, t: torch.tensor(np.asarray(x), dtype=t, device=cuda_device)  # noqa: E731
    cached, new, table, ring = (to(x, torch.int32) for x in case[:4])
    span, batch = to(case[4], torch.int64), len(case[0])
    slots = torch.full((rows + 2,), 77, dtype=torch.int64, device=cuda_device)
    positions, cu, lens = (torch.full((n + 2,), 77, dtype=torch.int32, device=cuda_device)
                           for n in (rows, batch + 1, batch))
    after = torch.empty(2, dtype=torch.int64, device=cuda_device)
    launcher("tm_build_block_tables")(0, packer(TmBlockTablesParams)(
        cached.data_ptr(), new.data_ptr(), table.data_ptr(), table.stride(0), table.shape[1], ring.data_ptr(),
        ring.numel(), span.data_ptr(), batch, page, rows, slots[1:].data_ptr(), positions[1:].data_ptr(),
        cu[1:].data_ptr(), lens[1:].data_ptr(), after.data_ptr()))
    ref = ora.build_block_tables(*case, page, rows)
    for got, want in zip((slots, positions, cu, lens), ref):
        got = got.cpu().numpy()
        assert np.array_equal(got[1:-1], want) and got[0] == got[-1] == 77
    assert np.array_equal(after.cpu().numpy(), ref[4]) and np.array_equal(table.cpu().numpy(), ref[5])


def test_release_of_many_long_requests(cuda_device):
    from tilemix_b200.attention.kv4 import release_pages

    page, batch = 16, 700
    rng = np.random.default_rng(11)
    lens = rng.integers(0, 5000, batch)
    lens[5], lens[600] = 131072, 0
    held = -(-lens // page)
    free, capacity = 1000, int(held.sum()) + 1000
    order = rng.permutation(capacity).astype(np.int32)
    table = np.full((batch, int(held.max()) + 1), -1, dtype=np.int32)
    at = free
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    done = rng.random(batch) < 0.5
    done[5] = True
    head = 3 * capacity - 500  # the free entries wrap, and so do those that come back
    ring = np.full(capacity, -7, dtype=np.int32)
    ring[(head + np.arange(free)) % capacity] = order[:free]
    to = lambda x, t: torch.tensor(x, dtype=t, device=cuda_device)  # noqa: E731
    args = [to(lens, torch.int32), to(done, torch.bool), to(table, torch.int32), to(ring, torch.int32),
            to([head, head + free], torch.int64)]
    release_pages(*args, page_size=page)
    back = np.concatenate([table[b, :held[b]] for b in range(batch) if done[b]])
    ring[(head + free + np.arange(len(back))) % capacity] = back
    table[done] = -1
    lens[done] = 0
    for got, want in zip(args, (lens, done, table, ring, [head, head + free + len(back)])):
        assert np.array_equal(got.cpu().numpy(), want)
