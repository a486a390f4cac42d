"""coda_paged_append and coda_paged_attn through the C ABI against plain 64-bit forms on the CPU."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from coda_amd import _lib  # noqa: E402

DEV = "cuda"
BF, F8, F64 = torch.bfloat16, torch.float8_e4m3fn, torch.float64
D = 128
HALF = {BF: 2.0 ** -8, F8: 2.0 ** -4}      # half a step of the stored type, relative to the value
F8_TINY = 2.0 ** -10                       # half a step of e4m3 below its smallest normal number


def _s():
    return torch.cuda.current_stream().cuda_stream


class Batch:
    """A ragged batch over a paged cache, on the CPU: `lens` new tokens behind `past` positions each."""

    def __init__(self, lens, past, page, n_q, n_kv, cache="bf16", seed=0, spare_rows=0, spare_pages=3, row_pad=0, page_pad=0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.past, self.page, self.n_q, self.n_kv = list(lens), list(past), page, n_q, n_kv
        self.B, self.f8 = len(lens), cache == "e4m3"
        self.total = [p + n for p, n in zip(past, lens)]
        self.starts = [0]
        for n in lens:
            self.starts.append(self.starts[-1] + n)
        self.T = self.starts[-1] + spare_rows             # rows behind the last sequence
        self.max_pages = max(1, -(-max(self.total) // page)) + 1
        used = [-(-t // page) for t in self.total]
        self.num_pages = sum(used) + spare_pages
        order = torch.randperm(self.num_pages, generator=g).to(torch.int32)
        self.table = torch.full((self.B, self.max_pages), 2 ** 30, dtype=torch.int32)       # unused entries: not a page
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = order[at:at + u]
            at += u
        self.k_scale, self.v_scale = (1 / 32, 1 / 64) if self.f8 else (1.0, 1.0)
        # pages lie page_pad elements apart, rows of q / qkv row_pad elements
        self.page_stride = n_kv * page * D + page_pad
        shape = (self.num_pages, self.page_stride)
        self.g = g
        if self.f8:
            self.k = (torch.randn(shape, generator=g) * 48).to(F8)
            self.v = (torch.randn(shape, generator=g) * 64).to(F8)
        else:
            self.k = (torch.randn(shape, generator=g) * 1.5).to(BF)
            self.v = torch.randn(shape, generator=g).to(BF)
        self.row_pad = row_pad
        self.q = (torch.randn(self.T, n_q * D + row_pad, generator=g) * 1.5).to(BF)
        self.seq_start = torch.tensor(self.starts, dtype=torch.int32)
        self.pos0 = torch.tensor(past, dtype=torch.int32)
        self.kv_len = torch.tensor(self.total, dtype=torch.int32)

    def pages(self, cache):
        """[num_pages, n_kv, page, 128] of the cache or of a view of it (the bytes of a bf16 cache: 256 a row)."""
        d = 2 * D if cache.dtype == torch.uint8 and not self.f8 else D
        return cache[:, :self.n_kv * self.page * d].view(self.num_pages, self.n_kv, self.page, d)

    def keys(self, cache, b, scale, n=None):
        """Keys 0 .. n-1 of sequence b: [n, n_kv, 128] in 64 bits, and which of them are on a page that is there."""
        n = self.total[b] if n is None else n
        at = torch.arange(n)
        row = self.table[b].long()[at // self.page]
        there = (row >= 0) & (row < self.num_pages)
        x = self.pages(cache.view(torch.uint8) if self.f8 else cache)[row.clamp(0, self.num_pages - 1), :, at % self.page]
        return (x.contiguous().view(F8) if self.f8 else x).to(F64) * scale, there


def attn(b, mask=0, scale=1 / math.sqrt(D), max_kv=None, dev=None, out=None, ws=None, stream=None):
    """One call; `dev`: tensors that are on the GPU already.  Returns the output on the GPU, NaN where nothing was written."""
    d = dev or {n: getattr(b, n).to(DEV) for n in ("q", "k", "v", "table", "seq_start", "pos0", "kv_len")}
    max_kv = max(b.total) if max_kv is None else max_kv
    if out is None:
        out = torch.full((b.T, b.n_q * D + b.row_pad), float("nan"), device=DEV, dtype=BF)
    size = _lib.load().coda_paged_attn_workspace_bytes(b.T, b.B, max_kv, b.n_q, b.n_kv)
    if ws is None:
        ws = torch.full((max(size, 16),), 255, device=DEV, dtype=torch.uint8)               # NaN patterns
    _lib.call("coda_paged_attn", d["q"].data_ptr(), d["q"].stride(0), out.data_ptr(), out.stride(0), d["seq_start"].data_ptr(),
              d["pos0"].data_ptr(), d["kv_len"].data_ptr(), b.B, b.T, d["table"].data_ptr(), d["table"].stride(0), b.max_pages,
              d["k"].data_ptr(), d["v"].data_ptr(), b.page_stride, b.num_pages, b.page, int(b.f8), b.k_scale, b.v_scale, max_kv, b.n_q,
              b.n_kv, scale, mask, ws.data_ptr(), size, stream or _s())
    if stream is None and dev is None:
        torch.cuda.synchronize()
    b.keep = (d, ws)
    return out


def attn_ref(b, mask=0, scale=1 / math.sqrt(D), max_kv=None):
    """(output, sum_j p_j |v_j|, bound on |score| rounding) in 64 bits; rows of no sequence are NaN."""
    out = torch.full((b.T, b.n_q, D), float("nan"), dtype=F64)
    mag, ds = torch.zeros_like(out), torch.zeros(b.T, b.n_q, 1, dtype=F64)
    for i, n in enumerate(b.lens):
        if not n:
            continue
        kv = min(max(int(b.kv_len[i]), 0), max(b.total) if max_kv is None else max_kv)
        k, there = b.keys(b.k, i, b.k_scale, kv)
        v, _ = b.keys(b.v, i, b.v_scale, kv)
        rows = slice(b.starts[i], b.starts[i + 1])
        q = b.q[rows, :b.n_q * D].to(F64).view(n, b.n_q, D)
        pos = int(b.pos0[i]) + torch.arange(n)
        lim = torch.full((n,), kv) if not mask else torch.minimum(torch.tensor(kv), (pos // mask + 1) * mask)
        seen = (torch.arange(kv)[None, :] < lim[:, None]) & there[None, :]
        for h in range(b.n_q):
            kh, vh = k[:, h // (b.n_q // b.n_kv)], v[:, h // (b.n_q // b.n_kv)]
            # keys that a row does not see are left out of its sums, not multiplied by zero
            z = torch.where(seen, q[:, h] @ torch.where(there[:, None], kh, 0.0).nan_to_num(0, 0, 0).t() * scale, -math.inf)
            p = torch.softmax(z, -1).nan_to_num(0.0)                            # rows that see nothing: zeros
            out[rows, h] = p @ vh.nan_to_num(0, 0, 0) if kv else torch.zeros(n, D, dtype=F64)
            mag[rows, h] = p @ vh.nan_to_num(0, 0, 0).abs() if kv else 0.0
            ds[rows, h, 0] = scale * q[:, h].norm(dim=-1) * (kh.nan_to_num(0, 0, 0).norm(dim=-1).max() if kv else 0.0)
    return out.view(b.T, -1), mag.view(b.T, -1), ds.expand(-1, -1, D).reshape(b.T, -1)


def check(out, b, **kw):
    """|out - ref| <= 2^-8 |ref| (the bf16 result) + 2 (2^-8 + ds) sum p |v|: every weight is off by at most half a bf16 step
    (2^-8) and by exp of its score's error, numerator and denominator both (hence 2); a score is a sum of 128 products in fp32,
    off by at most 128 * 2^-24 |q| |k| scale, its exponential by 2^-20 (the device's exp2 and the fp32 running sums)."""
    ref, mag, ds = attn_ref(b, **kw)
    got = out[:, :b.n_q * D].to(F64).cpu()
    n = b.starts[-1]
    err = (got[:n] - ref[:n]).abs()
    tol = 2.0 ** -8 * ref[:n].abs() + 2 * (2.0 ** -8 + 128 * 2.0 ** -24 * ds[:n] + 2.0 ** -20) * mag[:n] + 1e-30
    assert torch.isfinite(got[:n]).all()
    assert (err <= tol).all(), f"worst {(err / tol).max()} of the bound"
    # typical size: the roundings of one output are independent, so the whole is far inside the sum of bounds
    if ref[:n].norm() > 0:
        assert err.norm() / ref[:n].norm() < 2.0 ** -8
    assert torch.isnan(out[n:]).all(), "rows behind the last sequence were written"
    assert torch.isnan(out[:, b.n_q * D:]).all(), "columns behind the last head were written"


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [1, 8, 16, 24, 64, 100])
@pytest.mark.parametrize("lens,past,n_q,n_kv", [
    ([1], [0], 2, 1),                                       # a first token: one key
    ([1, 1, 1], [31, 32, 200], 16, 8),                      # single tokens around a tile's edge
    ([0, 5, 0, 1, 0], [3, 60, 0, 127, 9], 6, 2),            # sequences without a row, g = 3
    ([32, 32], [96, 17], 16, 8),                            # denoise blocks: 64 rows
    ([40, 3], [0, 300], 16, 8),                             # two tiles of 32 rows and a partial one
    ([130, 1, 77], [5, 64, 0], 16, 8),                      # past 128 rows, partial tiles
    ([300], [129], 12, 4),
])
def test_attention(lens, past, n_q, n_kv, page, cache):
    b = Batch(lens, past, page, n_q, n_kv, cache, seed=len(lens) * 100 + page, spare_rows=2, row_pad=8, page_pad=16)
    for mask in (0, 1, 32):
        check(attn(b, mask), b, mask=mask)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("g,n", [(1, 1), (2, 1), (7, 1), (16, 1), (33, 1), (16, 5), (16, 20), (1, 100), (5, 70)])
def test_attention_head_groups(g, n, cache):
    b = Batch([n, max(1, n // 2)], [50, 7], 16, g, 1, cache, seed=g)
    for mask in (0, 1):
        check(attn(b, mask), b, mask=mask)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("lens,past", [([1], [5000]), ([1, 1, 1], [3000, 10, 1700]), ([20, 1], [2500, 900]), ([60, 2], [4000, 4]),
                                       ([200], [2000]), ([300], [4000]), ([20] * 13, [2000 - 150 * i for i in range(13)])])
def test_attention_ranges_of_keys(lens, past, cache):
    """Few rows over many keys: the keys are cut into ranges and joined; short sequences of the batch have one range.  The last two: more
    rows and ranges than are joined in one step."""
    b = Batch(lens, past, 32, 4, 2, cache, seed=5)
    assert _lib.load().coda_paged_attn_workspace_bytes(b.T, b.B, max(b.total), 4, 2) > 0
    for mask in (0, 1):
        check(attn(b, mask), b, mask=mask)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [16, 10])
@pytest.mark.parametrize("lens,past,n_q,n_kv,max_kv", [
    ([200], [500], 320, 40, 700),                           # many heads: tiles enough without ranges
    ([60, 40], [3000, 20], 64, 2, 40000),                   # few: ranges of keys, out of a long bound
])
def test_attention_widest_tiles(lens, past, n_q, n_kv, max_kv, page, cache):
    """More than 1536 rows a sequence and key/value head: 256-row tiles."""
    b = Batch(lens, past, page, n_q, n_kv, cache, seed=6, spare_rows=1)
    pages = -(-max_kv // page)
    b.table = torch.cat((b.table, torch.full((b.B, pages), -1, dtype=torch.int32)), 1)
    b.max_pages += pages
    assert (_lib.load().coda_paged_attn_workspace_bytes(b.T, b.B, max_kv, n_q, n_kv) > 0) == (n_kv == 2)
    for mask in (0, 1, 32):
        check(attn(b, mask, max_kv=max_kv), b, mask=mask)
    # NaN in the last key's V, which under the causal mask only the last token sees
    last = b.total[0] - 1
    clean = attn(b, 1, max_kv=max_kv).clone()
    v = b.pages(b.v.view(torch.uint8) if b.f8 else b.v.view(torch.int16))
    v[int(b.table[0, last // page]), 0, last % page, 77] = 0x7f if b.f8 else torch.tensor(float("nan"), dtype=BF).view(torch.int16)
    out, row = attn(b, 1, max_kv=max_kv), b.starts[1] - 1
    hit = torch.zeros(b.T, n_q, D, dtype=torch.bool, device=DEV)
    hit[row, :n_q // n_kv, 77] = True
    hit = hit.view(b.T, -1)
    hit[b.starts[-1]:] = True                               # rows of no sequence: never written
    assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("B,past", [(150, 40), (300, 40), (300, 3000)])
def test_attention_many_sequences(B, past):
    """More sequences than one step of the search covers, many of them without a row; the last case cuts the keys into ranges."""
    lens = [(i * 7) % 3 for i in range(B)]
    b = Batch(lens, [(i * 1301) % past for i in range(B)], 8, 2, 1, seed=8)
    for mask in (0, 1):
        check(attn(b, mask), b, mask=mask)


@pytest.mark.parametrize("lens", [[1, 1, 1], [40, 3, 20], [70, 9, 9], [200, 90, 30]])
def test_attention_no_keys_beside_many(lens):
    """Ranges of keys, and sequences of the same call with none, one or no page."""
    b = Batch(lens, [4000, 10, 900], 16, 4, 2, seed=13)
    b.kv_len[1] = 0
    b.table[2] = -1
    for mask in (0, 1):
        out = attn(b, mask)
        check(out, b, mask=mask)
        assert (out[b.starts[1]:b.starts[3]] == 0).all()
    b.kv_len[0] = 1
    check(attn(b, 0, max_kv=max(b.total)), b, mask=0)


def test_attention_rows_before_the_first_sequence():
    b = Batch([4, 0, 70], [30, 3, 10], 16, 4, 2, seed=9, spare_rows=5)
    want = attn(b, 1).clone()
    b.seq_start += 3
    b.q = torch.cat((b.q[-3:], b.q[:-3]))
    out = attn(b, 1)
    assert torch.isnan(out[:3]).all() and torch.equal(out[3:77], want[:74]) and torch.isnan(out[77:]).all()


@pytest.mark.parametrize("starts", [[0, 90, 40, 60], [50, 10, 10, 90], [-7, 20, 200, 30], [300, 300, 300, 300], [-1, -1, -1, -1]])
def test_attention_starts_that_make_no_sense(starts):
    """Starts that decrease or leave [0, T]: rows come out wrong or not at all, and nothing else is touched."""
    b = Batch([30, 30, 30], [20, 70, 40], 16, 4, 2, seed=10)
    b.seq_start = torch.tensor(starts, dtype=torch.int32)
    guard = torch.full((b.T + 64, b.n_q * D), 7.0, device=DEV, dtype=BF)
    attn(b, 1, out=guard[32:32 + b.T])
    assert (guard[:32] == 7).all() and (guard[32 + b.T:] == 7).all()
    qkv, qw, kw = inputs(b)
    cos, sin = rope(300)
    _, k, v = append(b, qkv, qw, kw, cos, sin)               # positions that follow from such starts may have no page: skipped
    assert torch.isfinite(k.float()).all() and torch.isfinite(v.float()).all()


@pytest.mark.parametrize("page", [16, 10])
@pytest.mark.parametrize("lens", [[1, 1], [30, 2], [60, 64], [150, 9], [90, 200]])
def test_attention_lengths_and_bad_pages(lens, page):
    """kv_len of zero, negative or beyond max_kv; page numbers that are no pages.  A row that sees nothing gets zeros."""
    b = Batch(lens, [100, 100], page, 4, 2, seed=11)
    b.table[0, 2] = -1
    b.table[0, 4] = b.num_pages
    b.table[0, 5] = -2 ** 31
    check(attn(b, 0), b, mask=0)
    check(attn(b, 1, max_kv=70), b, mask=1, max_kv=70)      # kv_len beyond max_kv
    b.kv_len[1] = -5
    out = attn(b, 0)
    check(out, b, mask=0)
    assert (out[b.starts[1]:b.starts[2]] == 0).all()
    b.kv_len[0] = 0
    b.kv_len[1] = 1
    check(attn(b, 0), b, mask=0)
    out = attn(b, 0, max_kv=0)
    assert (out[:b.starts[-1]] == 0).all()
    # every page gone
    b.kv_len[:] = torch.tensor(b.total)
    b.table[:] = -1
    out = attn(b, 0)
    assert (out[:b.starts[-1]] == 0).all()


@pytest.mark.parametrize("cache,bad", [("bf16", float("inf")), ("bf16", float("-inf")), ("bf16", float("nan")), ("e4m3", float("nan"))])
@pytest.mark.parametrize("lens,past", [([3], [40]), ([20, 9], [64, 10]), ([32, 30], [40, 41]), ([60, 2], [13, 90]), ([140], [77]),
                                       ([90, 200], [13, 41])])
def test_attention_nonfinite_where_nobody_looks(lens, past, bad, cache):
    """Infinities and NaN in slots behind the sequence and on unused pages; and in keys that only LATER tokens see."""
    b = Batch(lens, past, 16, 4, 2, cache, seed=21)
    clean = {m: attn(b, m).clone() for m in (0, 1)}
    live = torch.zeros(b.num_pages, b.page, dtype=torch.bool)
    for i, t in enumerate(b.total):
        at = torch.arange(t)
        live[b.table[i].long()[at // b.page], at % b.page] = True
    value = 0x7f if b.f8 else torch.tensor(bad, dtype=BF).view(torch.int16)
    k, v = (b.pages(c.view(torch.uint8) if b.f8 else c.view(torch.int16)) for c in (b.k, b.v))
    k.permute(0, 2, 1, 3)[~live] = value
    v.permute(0, 2, 1, 3)[~live] = value
    for m in (0, 1):
        out = attn(b, m)
        assert torch.equal(out[:b.starts[-1]], clean[m][:b.starts[-1]])
    # the last key of sequence 0, one feature of V and all of K: with the causal mask only the last token sees it
    last = b.total[0] - 1
    page, slot = int(b.table[0, last // b.page]), last % b.page
    v[page, 0, slot, 77] = value
    out = attn(b, 1)
    row = b.starts[1] - 1
    others = torch.tensor([r for r in range(b.starts[-1]) if r != row])
    assert torch.equal(out[others], clean[1][others])
    heads = out[row].view(b.n_q, D)
    assert not torch.isfinite(heads[:2, 77]).any() and torch.isfinite(heads[2:]).all()
    keep = [d for d in range(D) if d != 77]
    assert torch.equal(heads[:, keep], clean[1][row].view(b.n_q, D)[:, keep])
    k[page, 1, slot, 5] = 0x7f if b.f8 else torch.tensor(float("nan"), dtype=BF).view(torch.int16)
    out = attn(b, 1)
    assert torch.equal(out[others], clean[1][others])
    assert torch.isnan(out[row].view(b.n_q, D)[2:]).all()


def test_attention_large_scores():
    """Scores of many hundred: the running maximum moves by more than fp32's exponent range from tile to tile."""
    b = Batch([2, 40], [500, 300], 16, 4, 2, seed=31)
    b.q *= 30
    for mask in (0, 1):
        check(attn(b, mask), b, mask=mask)


@pytest.mark.parametrize("lens,past", [([1], [4000]), ([32], [300]), ([200], [60])])
def test_attention_same_bits_every_time(lens, past):
    b = Batch(lens, past, 16, 16, 8, seed=41)
    first = attn(b, 1).clone()
    for _ in range(3):
        assert torch.equal(attn(b, 1)[:b.T], first)


@pytest.mark.parametrize("page", [16, 10])
def test_far_pages(page):
    """Pages whose offset passes 2^32 bytes, read and written."""
    if torch.cuda.mem_get_info()[0] < 50 << 30:
        pytest.skip("needs 50 GB")
    b = Batch([1, 40], [70, 90], page, 4, 2, seed=51)
    far = (5 << 30) // 2 // 4                                # elements between pages: page 4 starts at 5 GiB
    far -= far % 8
    d = {n: getattr(b, n).to(DEV) for n in ("q", "table", "seq_start", "pos0", "kv_len")}
    spots = 5                                                # the sequences share five pages, wherever those are
    inside = (b.table >= 0) & (b.table < b.num_pages)
    b.table[inside] %= spots
    pool_k = torch.zeros(4 * far + b.page_stride, dtype=BF, device=DEV)
    pool_v = torch.zeros_like(pool_k)
    for p in range(spots):
        pool_k[p * far:p * far + b.page_stride] = b.k[p].to(DEV)
        pool_v[p * far:p * far + b.page_stride] = b.v[p].to(DEV)
    table = b.table
    want = attn(b, 1).clone()
    check(want, b, mask=1)
    d["k"], d["v"], d["table"] = pool_k, pool_v, table.to(DEV)
    stride, b.page_stride, pages, b.num_pages = b.page_stride, far, b.num_pages, spots
    got = attn(b, 1, dev=d)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    # one new token on the page behind 2^32 bytes: only its slot changes
    g = Batch([1], [0], page, 4, 2, seed=52)
    g.table[0, 0], g.num_pages, g.page_stride = 4, spots, far
    qkv, qw, kw = inputs(g)
    cos, sin = rope(1)
    near_b = Batch([1], [0], page, 4, 2, seed=52)
    _, k_near, v_near = append(near_b, qkv, qw, kw, cos, sin)
    before = pool_k[4 * far:].clone(), pool_v[4 * far:].clone()
    d = {"k": pool_k, "v": pool_v, "table": g.table.to(DEV), "seq_start": g.seq_start.to(DEV), "pos0": g.pos0.to(DEV)}
    append(g, qkv, qw, kw, cos, sin, dev=d, fetch=False)
    for pool, old, new in ((pool_k, before[0], k_near), (pool_v, before[1], v_near)):
        got = pool[4 * far:].view(2, page, D).cpu()
        assert torch.equal(got[:, 0], near_b.pages(new)[int(near_b.table[0, 0]), :, 0])
        assert torch.equal(got[:, 1:], old.view(2, page, D).cpu()[:, 1:])
    assert not pool_k[:4 * far].view(4, far)[:, b.n_kv * page * D:].any()
    b.page_stride, b.num_pages = stride, pages


def test_attention_on_another_stream_and_in_a_graph():
    b = Batch([1, 33, 2], [3000, 40, 700], 16, 8, 4, seed=61)
    want = attn(b, 1).clone()
    d = b.keep[0]
    out, ws = torch.full_like(want, float("nan")), b.keep[1]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attn(b, 1, dev=d, out=out, ws=ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn(b, 1, dev=d, out=out, ws=ws, stream=torch.cuda.current_stream().cuda_stream)
    for n in (0, 1, 2):
        out.fill_(float("nan"))
        b.kv_len[0] = b.total[0] - 900 * n                  # the lengths are read when the graph runs
        d["kv_len"].copy_(b.kv_len)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, attn(b, 1, max_kv=max(b.total)))


# ------------------------------------------------------------------------------------------------ append
def append(b, qkv, qw, kw, cos, sin, flags=0, in_place=False, eps=1e-6, dev=None, fetch=True):
    d = dev or {n: getattr(b, n).to(DEV) for n in ("k", "v", "table", "seq_start", "pos0")}
    x = qkv.to(DEV).clone()
    q_out = x if in_place else torch.full((b.T, b.n_q * D + 16), float("nan"), device=DEV, dtype=BF)
    w = [None if t is None else t.to(DEV) for t in (qw, kw)]
    c = [cos.to(DEV), sin.to(DEV)]
    _lib.call("coda_paged_append", x.data_ptr(), x.stride(0), q_out.data_ptr(), q_out.stride(0), *[None if t is None else t.data_ptr() for t in w],
              c[0].data_ptr(), c[1].data_ptr(), cos.shape[0], d["seq_start"].data_ptr(), d["pos0"].data_ptr(), b.B, b.T,
              d["table"].data_ptr(), d["table"].stride(0), b.max_pages, d["k"].data_ptr(), d["v"].data_ptr(), b.page_stride, b.num_pages,
              b.page, int(b.f8), b.k_scale, b.v_scale, b.n_q, b.n_kv, eps, flags, _s())
    torch.cuda.synchronize()
    if not in_place:
        assert torch.equal(x.cpu().view(torch.int16), qkv.view(torch.int16))
    return (q_out.cpu(), d["k"].cpu(), d["v"].cpu()) if fetch else None


def rope(n, theta=1e6):
    ang = torch.arange(n, dtype=F64)[:, None] / theta ** (torch.arange(0, D, 2, dtype=F64) / D)[None, :]
    ang = torch.cat((ang, ang), -1)
    return ang.cos().to(BF), ang.sin().to(BF)


def inputs(b, seed=1, norm=True):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(b.T, (b.n_q + 2 * b.n_kv) * D + 8, generator=g).to(BF)
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(BF) for _ in range(2)] if norm else [None, None]
    return qkv, w[0], w[1]


def turned(x, w, cos, sin, eps):
    """[n, heads, 128] in 64 bits: normalised, rotated; and the sum of magnitudes of the rotation's two products."""
    n = x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.to(F64)
    lo, hi = n[..., :64], n[..., 64:]
    c, s = cos.to(F64)[:, None], sin.to(F64)[:, None]
    half = torch.cat((-hi, lo), -1)
    return n * c + half * s, (n * c).abs() + (half * s).abs()


def near(got, want, mag, dtype):
    """One rounding to the stored type, and fp32 arithmetic of 128 + 8 roundings before it."""
    tol = HALF[dtype] * want.abs() + (136 * 2.0 ** -24) * mag * (1 + HALF[dtype]) + (F8_TINY if dtype is F8 else 1e-30)
    err = (got.to(F64) - want).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max()} of the bound"


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("lens,past,n_q,n_kv,norm", [
    ([1], [0], 16, 8, True), ([1, 1, 1], [15, 16, 200], 16, 8, True), ([0, 9, 0, 2], [1, 14, 0, 40], 6, 2, True),
    ([33, 70], [3, 0], 5, 5, False), ([400], [0], 16, 8, True), ([3, 4], [2, 9], 1, 1, True), ([2], [6], 40, 8, True)])
def test_append(lens, past, n_q, n_kv, norm, page, cache):
    b = Batch(lens, past, page, n_q, n_kv, cache, seed=2, spare_rows=3, page_pad=32)
    qkv, qw, kw = inputs(b, norm=norm)
    cos, sin = rope(max(b.total))
    q_out, k, v = append(b, qkv, qw, kw, cos, sin)
    touched = torch.zeros(b.num_pages, b.page, dtype=torch.bool)
    stored = F8 if b.f8 else BF
    for i, n in enumerate(b.lens):
        rows = slice(b.starts[i], b.starts[i + 1])
        pos = past[i] + torch.arange(n)
        x = qkv[rows, :(n_q + 2 * n_kv) * D].to(F64).view(n, n_q + 2 * n_kv, D)
        q, mag = turned(x[:, :n_q], qw, cos[pos], sin[pos], 1e-6)
        near(q_out[rows, :n_q * D].view(n, n_q, D), q, mag, BF)
        kk, mag = turned(x[:, n_q:n_q + n_kv], kw, cos[pos], sin[pos], 1e-6)
        page_no, slot = b.table[i].long()[pos // page], pos % page
        got_k = b.pages(k.view(torch.uint8) if b.f8 else k)[page_no, :, slot].contiguous().view(stored)
        got_v = b.pages(v.view(torch.uint8) if b.f8 else v)[page_no, :, slot].contiguous().view(stored)
        near(got_k, (kk / b.k_scale).clamp(-448, 448) if b.f8 else kk, mag / b.k_scale, stored)
        vv = x[:, n_q + n_kv:] / b.v_scale
        if b.f8:
            near(got_v, vv.clamp(-448, 448), vv.abs(), F8)
        else:
            assert torch.equal(got_v, x[:, n_q + n_kv:].to(BF))
        touched[page_no, slot] = True
    # every other slot, the gaps between pages, rows of no sequence and columns behind the heads: as they were
    for new, old in ((k, b.k), (v, b.v)):
        new, old = new.view(torch.uint8), old.view(torch.uint8)
        same = b.pages(new).permute(0, 2, 1, 3)[~touched], b.pages(old).permute(0, 2, 1, 3)[~touched]
        assert torch.equal(*same)
        size = b.n_kv * b.page * D * (1 if b.f8 else 2)
        assert torch.equal(new[:, size:], old[:, size:])
    assert torch.isnan(q_out[b.starts[-1]:]).all() and torch.isnan(q_out[:, n_q * D:]).all()


def test_append_in_place_and_stepwise_bits():
    """In place equals out of place; the stepwise form has the bits of coda_qknorm_rope."""
    b = Batch([5, 5, 5], [0, 0, 0], 4, 16, 8, seed=3)
    qkv, qw, kw = inputs(b)
    cos, sin = rope(5)
    for flags in (0, _lib.APPEND_STEPWISE):
        far = append(b, qkv, qw, kw, cos, sin, flags)
        here = append(b, qkv, qw, kw, cos, sin, flags, in_place=True)
        assert torch.equal(far[0][:, :16 * D], here[0][:, :16 * D])
        assert torch.equal(here[0][:, 16 * D:], qkv[:, 16 * D:])
        assert torch.equal(far[1], here[1]) and torch.equal(far[2], here[2])
    x = qkv.to(DEV).clone()
    w = [t.to(DEV) for t in (qw, kw, cos, sin)]
    _lib.call("coda_qknorm_rope", x.data_ptr(), x.stride(0), *[t.data_ptr() for t in w], 15, 5, 16, 8, 1e-6, _s())
    torch.cuda.synchronize()
    x = x.cpu()
    q_out, k, v = append(b, qkv, qw, kw, cos, sin, _lib.APPEND_STEPWISE)
    assert torch.equal(q_out[:, :16 * D], x[:, :16 * D])
    for i in range(3):
        pos = torch.arange(5)
        page_no, slot = b.table[i].long()[pos // 4], pos % 4
        rows = x[5 * i:5 * i + 5]
        assert torch.equal(b.pages(k)[page_no, :, slot].reshape(5, -1), rows[:, 16 * D:24 * D])
        assert torch.equal(b.pages(v)[page_no, :, slot].reshape(5, -1), rows[:, 24 * D:32 * D])


def test_append_thousands_of_sequences():
    """Three steps of the search for a token's sequence; almost all sequences have no row."""
    B = 5000
    lens = [1 if i % 71 == 3 else 0 for i in range(B)]
    b = Batch(lens, [i % 5 for i in range(B)], 4, 2, 1, seed=12)
    qkv, qw, kw = inputs(b)
    cos, sin = rope(8)
    q_out, k, v = append(b, qkv, qw, kw, cos, sin)
    for i in [i for i in range(B) if lens[i]]:
        row, pos = b.starts[i], b.past[i]
        x = qkv[row:row + 1, :4 * D].to(F64).view(1, 4, D)
        q, mag = turned(x[:, :2], qw, cos[pos:pos + 1], sin[pos:pos + 1], 1e-6)
        near(q_out[row:row + 1, :2 * D].view(1, 2, D), q, mag, BF)
        assert torch.equal(b.pages(v)[int(b.table[i, pos // 4]), 0, pos % 4], qkv[row, 3 * D:4 * D])


def test_append_skips_what_has_no_place():
    """Positions before 0 and behind the rotary table: nothing at all; a page that is not there: the q row only."""
    b = Batch([4, 4, 4], [0, 8, 4], 4, 2, 1, seed=4)
    qkv, qw, kw = inputs(b)
    cos, sin = rope(10)                                     # sequence 1 is at 8 .. 11: two tokens have no rotary row
    b.pos0[0] = -2                                          # sequence 0 at -2 .. 1: two tokens before the start
    b.table[2, 1] = -1                                      # sequence 2's page is gone
    q_out, k, v = append(b, qkv, qw, kw, cos, sin)
    written = [not torch.isnan(q_out[r, :2 * D]).any() for r in range(12)]
    assert written == [False, False, True, True, True, True, False, False, True, True, True, True]
    slots = {(int(b.table[0, 0]), 0), (int(b.table[0, 0]), 1), (int(b.table[1, 2]), 0), (int(b.table[1, 2]), 1)}
    for new, old in ((k, b.k), (v, b.v)):
        changed = (b.pages(new) != b.pages(old)).any(-1).any(1)
        assert {tuple(x) for x in changed.nonzero().tolist()} == slots


def test_append_e4m3_saturates_and_keeps_nan():
    b = Batch([3], [0], 16, 1, 1, "e4m3", seed=6)
    qkv, _, _ = inputs(b, norm=False)
    cos, sin = torch.ones(16, D, dtype=BF), torch.zeros(16, D, dtype=BF)
    qkv[0, 2 * D], qkv[0, 2 * D + 1], qkv[0, 2 * D + 2] = 1e5, -1e5, float("nan")
    qkv[1, 2 * D], qkv[1, 2 * D + 1] = float("inf"), float("-inf")
    qkv[2, D:2 * D] = 0
    qkv[2, D], qkv[2, D + 1] = 1e30, -7.5                   # the key keeps its signs and zeros, clamped
    _, k, v = append(b, qkv, None, None, cos, sin)
    page = int(b.table[0, 0])
    got = b.pages(v.view(torch.uint8))[page, 0].contiguous().view(F8).float()
    assert got[0, 0] == 448 and got[0, 1] == -448 and torch.isnan(got[0, 2]) and got[1, 0] == 448 and got[1, 1] == -448
    got = b.pages(k.view(torch.uint8))[page, 0].contiguous().view(F8).float()
    assert got[2, 0] == 448 and got[2, 1] == -240 and (got[2, 2:] == 0).all()


@pytest.mark.parametrize("mask", [1, 64])
@pytest.mark.parametrize("B", [2, 9, 16, 17])
def test_attention_tile_order(B, mask):
    """Long prompts of very different lengths and pasts, masked: every tile of every sequence is done, whatever order they are taken
    in (up to 16 sequences longest first, more in sequence order)."""
    lens = [(i * 97) % 260 for i in range(B)]
    lens[0], lens[1] = 300, 131
    past = [(i * 211) % 500 for i in range(B)]
    b = Batch(lens, past, 64, 2, 1, seed=71)
    b.pos0[1] = -40                                          # the first 40 tokens see nothing
    check(attn(b, mask), b, mask=mask)
    b.pos0[0] = 10 ** 6                                      # far behind every key: all rows see all of them
    b.kv_len[2 % B] = 0
    check(attn(b, mask), b, mask=mask)


# ------------------------------------------------------------------------------------------------ how exact the weights are
def check_pair(out, b, **kw):
    """check() for weights that keep 16 bits: |out - ref| <= 2^-8 |ref| (the bf16 result) + 2 (2^-16 + ds + sums) sum p |v|.  A weight is
    a bf16 value and the bf16 value of its remainder: half a step of half a step, 2^-8 * 2^-8.  ds: a score is a sum of 128 products
    in fp32.  sums: two products a key, added up in fp32, and 2^-20 for the device's exp2.  Numerator and denominator, hence 2."""
    ref, mag, ds = attn_ref(b, **kw)
    n = b.starts[-1]
    got = out[:n, :b.n_q * D].to(F64).cpu()
    sums = 2 * max(b.total) * 2.0 ** -24 + 2.0 ** -20
    tol = 2.0 ** -8 * ref[:n].abs() + 2 * (2.0 ** -16 + 128 * 2.0 ** -24 * ds[:n] + sums) * mag[:n] * (1 + 2.0 ** -8) + 1e-30
    err = (got - ref[:n]).abs()
    bad = err > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outputs, worst {(err / tol).max()} of the bound, rows {bad.any(1).nonzero()[:4, 0].tolist()} .."


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [16, 10])
@pytest.mark.parametrize("lens,past,n_q,n_kv", [
    ([1, 1, 1], [40, 3, 17], 16, 8),                         # tiles of 16 rows
    ([16, 9], [24, 31], 6, 2),                               # of 32
    ([66, 60], [3, 10], 4, 2),                               # of 32, more than 64 rows a sequence
    ([100, 90], [10, 0], 4, 2),                              # of 128
    ([90], [430], 4, 2),                                     # of 128, keys in ranges
    ([300, 1, 1, 1], [0, 50, 7, 31], 16, 8),                 # of 128: single tokens beside a prompt
    ([200], [0], 320, 40),                                   # of 256
    ([1] * 9 + [120], [20 + i for i in range(9)] + [0], 16, 8),     # of 32: a prompt among single tokens
])
def test_attention_weights_keep_sixteen_bits(lens, past, n_q, n_kv, page, cache):
    """Whatever tiles a call is cut into and whatever else is in it.  Small queries: weights of like size, whose roundings would show."""
    b = Batch(lens, past, page, n_q, n_kv, cache, seed=81)
    b.q *= 0.4
    for mask in (0, 1):
        check_pair(attn(b, mask), b, mask=mask)


@pytest.mark.parametrize("seed", [1, 2, 3])
@pytest.mark.parametrize("lens,past", [([7], [60]), ([16, 2], [90, 10]), ([60, 3], [100, 20]), ([140], [77]), ([300, 9], [40, 600])])
def test_attention_unseen_keys_move_no_bit(lens, past, seed):
    """A key that only the last token of a sequence sees, with a score far above all others: every other row keeps its bits, also those
    that share a wave with it and its rescaling."""
    b = Batch(lens, past, 16, 4, 2, seed=90 + seed)
    clean = attn(b, 1).clone()
    last, row = b.total[0] - 1, b.starts[1] - 1
    q = b.q[row, :b.n_q * D].view(b.n_kv, b.n_q // b.n_kv, D)[:, 0]
    b.pages(b.k)[int(b.table[0, last // b.page]), :, last % b.page] = 8 * q         # a score of 8 |q|^2 / sqrt(128), about 200
    out = attn(b, 1)
    others = torch.tensor([r for r in range(b.starts[-1]) if r != row])
    assert not torch.equal(out[row], clean[row])
    assert torch.equal(out[others], clean[others])


def uncut(b):
    """No ranges of keys: no workspace."""
    return _lib.load().coda_paged_attn_workspace_bytes(b.T, b.B, max(b.total), b.n_q, b.n_kv) == 0


@pytest.mark.parametrize("mask", [1, 64])
@pytest.mark.parametrize("B,n_q,n_kv", [(1, 2, 1), (2, 2, 1), (9, 2, 1), (16, 2, 1), (17, 2, 1), (16, 32, 16), (17, 32, 16), (9, 32, 2)])
def test_attention_uncut_tile_order(B, n_q, n_kv, mask):
    """Masked prompts whose keys are not cut into ranges, of very different lengths and pasts: every tile of every sequence is done,
    whatever order they are taken in (up to 16 sequences longest first, more in sequence order).  The last: 256-row tiles."""
    lens = [(i * 97) % 260 for i in range(B)] if n_kv != 2 else [290 - 13 * i for i in range(B)]
    lens[0] = 300
    past = [(i * 211) % 200 for i in range(B)]
    b = Batch(lens, past, 64, n_q, n_kv, seed=73)
    assert uncut(b) and b.T * (n_q // n_kv) > 128 * B
    check(attn(b, mask), b, mask=mask)
    b.pos0[B - 1] = -40                                      # the first 40 tokens see nothing
    check(attn(b, mask), b, mask=mask)
    b.pos0[0] = 10 ** 6                                      # far behind every key: all rows see all of them
    b.kv_len[2 % B] = 0
    b.table[B // 2, 1] = -1
    check(attn(b, mask), b, mask=mask)


@pytest.mark.parametrize("starts", [[0, 300, 140, 220], [150, 10, 10, 450], [-7, 20, 900, 30], [900, 900, 900, 900], [-1, -1, -1, -1], [450, 0, 450, 0]])
@pytest.mark.parametrize("mask", [0, 1])
def test_attention_uncut_prompts_with_starts_that_make_no_sense(starts, mask):
    b = Batch([150, 150, 150], [20, 70, 40], 16, 4, 2, seed=10)
    assert uncut(b)
    b.seq_start = torch.tensor(starts, dtype=torch.int32)
    guard = torch.full((b.T + 64, b.n_q * D), 7.0, device=DEV, dtype=BF)
    attn(b, mask, out=guard[32:32 + b.T])
    assert (guard[:32] == 7).all() and (guard[32 + b.T:] == 7).all()


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("lens,past,later,n_q,n_kv,cut", [
    ([1, 1, 1], [40, 0, 17], [300, 2, 0], 16, 8, False),     # 16-row tiles
    ([1, 2], [1000, 30], [3000, 5], 4, 2, True),
    ([16, 9], [100, 31], [60, 200], 6, 2, False),            # 32
    ([32, 20], [1000, 64], [2000, 900], 4, 2, True),
    ([100, 90], [64, 0], [64, 300], 4, 2, False),            # 128
    ([64, 64], [1000, 300], [3000, 0], 8, 2, True),          # a block of 64 at 1000 of 4064 keys
    ([200, 130], [500, 1500], [2000, 100], 4, 2, True),
    ([200], [64], [300], 320, 40, False),                    # 256
    ([60, 40], [1000, 320], [2500, 600], 64, 2, True),
])
def test_attention_later_positions(lens, past, later, n_q, n_kv, cut, cache):
    """The denoiser's step in the middle of a sequence: keys behind the new tokens are in the cache.  Unmasked rows see them, masked ones
    those of their own block."""
    b = Batch(lens, [p + x for p, x in zip(past, later)], 16, n_q, n_kv, cache, seed=75, spare_rows=1)
    b.pos0 -= torch.tensor(later, dtype=torch.int32)
    assert uncut(b) != cut
    outs = {}
    for mask in (0, 1, 32, 64):
        outs[mask] = attn(b, mask)
        check(outs[mask], b, mask=mask)
    # what is not seen: keys from the end of the last token's block on
    for mask in (1, 64):
        d = {n: getattr(b, n).clone().to(DEV) for n in ("q", "k", "v", "table", "seq_start", "pos0", "kv_len")}
        d["kv_len"] = torch.minimum(b.kv_len, (b.pos0 + torch.tensor(lens, dtype=torch.int32) - 1) // mask * mask + mask).to(DEV)
        less = attn(b, mask, dev=d)
        torch.cuda.synchronize()
        n = b.starts[-1]
        # both within half a step of one value
        assert (less[:n].float() - outs[mask][:n].float()).norm() <= 2 * 2.0 ** -8 * outs[mask][:n].float().norm()


def test_attention_of_a_mixed_step_in_two_calls():
    """Prompts in front, single tokens behind: one call for each kind, the second with its rows, starts and page table from there on."""
    b = Batch([150, 90] + [1] * 6, [30, 0] + [100 + 90 * i for i in range(6)], 16, 16, 8, seed=77)
    check_pair(attn(b, 1), b, mask=1)
    d = {n: getattr(b, n).to(DEV) for n in ("q", "k", "v", "table", "seq_start", "pos0", "kv_len")}
    out, cut, row, T, B = torch.full((b.T, b.n_q * D), float("nan"), device=DEV, dtype=BF), 2, b.starts[2], b.T, b.B
    b.T, b.B = row, cut
    attn(b, 1, dev=d, out=out)
    first = b.keep
    late = {n: d[n][cut:] for n in ("table", "pos0", "kv_len")} | {"q": d["q"][row:], "seq_start": d["seq_start"][cut:] - row, "k": d["k"], "v": d["v"]}
    b.T, b.B = T - row, B - cut
    attn(b, 1, dev=late, out=out[row:])
    torch.cuda.synchronize()
    del first
    b.T, b.B = T, B
    check_pair(out, b, mask=1)
