"""coda_lora_bf16 through the C ABI against a plain 64-bit form on the CPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from coda_amd import _lib  # noqa: E402

DEV = "cuda"
BF, F64 = torch.bfloat16, torch.float64


def _s():
    return torch.cuda.current_stream().cuda_stream


class Case:
    def __init__(self, lens, adapters, K, N, rank, n=3, seed=0, spare=2, pad=0, scale=True):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.K, self.N, self.rank, self.n, self.B = list(lens), K, N, rank, n, len(lens)
        self.starts = [0]
        for m in lens:
            self.starts.append(self.starts[-1] + m)
        self.T, self.live = self.starts[-1] + spare, self.starts[-1]
        self.x = torch.randn(self.T, K + pad, generator=g).to(BF)
        self.r = torch.randn(self.T, N + pad, generator=g).to(BF)
        self.a = (torch.randn(n, rank, K, generator=g) * K ** -0.5).to(BF)
        self.b = (torch.randn(n, N, rank, generator=g) * rank ** -0.5).to(BF)
        self.scale = torch.rand(n, generator=g) * 2 - 0.5 if scale else None
        self.seq_start = torch.tensor(self.starts, dtype=torch.int32)
        self.adapter = torch.tensor(adapters, dtype=torch.int32)

    def device(self):
        return {k: None if getattr(self, k) is None else getattr(self, k).to(DEV) for k in ("x", "r", "a", "b", "scale", "seq_start", "adapter")}

    def call(self, d=None, out=None, in_place=False, ws=None, stream=None):
        d = d or self.device()
        if in_place:
            d["r"] = d["r"].clone()
            out = d["r"]
        if out is None:
            out = torch.full_like(d["r"], float("nan"))
        size = _lib.load().coda_lora_workspace_bytes(self.T, self.B, self.N, self.K, self.rank)
        if ws is None:
            ws = torch.full((max(size, 16),), 255, dtype=torch.uint8, device=DEV)       # NaN patterns
        _lib.call("coda_lora_bf16", d["x"].data_ptr(), d["x"].stride(0), d["a"].data_ptr(), d["b"].data_ptr(),
                  None if d["scale"] is None else d["scale"].data_ptr(), d["seq_start"].data_ptr(), d["adapter"].data_ptr(), self.B,
                  self.T, self.n, self.rank, d["r"].data_ptr(), d["r"].stride(0), out.data_ptr(), out.stride(0), self.N, self.K,
                  ws.data_ptr(), size, stream or _s())
        self.keep = (d, ws)
        return out

    def check(self, out):
        """The result's own rounding (2^-8), U's as a bf16 pair (2^-16 of |s u| |b|), and fp32 sums of K, then rank + 1 terms."""
        torch.cuda.synchronize()
        got = out[:self.live, :self.N].to(F64).cpu()
        want, tol = self.r[:self.live, :self.N].to(F64).clone(), torch.zeros(self.live, self.N, dtype=F64)
        for i, ad in enumerate(self.adapter.tolist()):
            rows = slice(self.starts[i], self.starts[i + 1])
            if not 0 <= ad < self.n:
                assert torch.equal(out[rows, :self.N].cpu(), self.r[rows, :self.N])
                continue
            s = 1.0 if self.scale is None else float(self.scale[ad])
            x, a, b = self.x[rows, :self.K].to(F64), self.a[ad].to(F64), self.b[ad].to(F64)
            want[rows] += s * (x @ a.t() @ b.t())
            mag_u = x.abs() @ a.abs().t()
            tol[rows] = abs(s) * (2.0 ** -16 + 2.0 ** -23) * ((x @ a.t()).abs() @ b.abs().t())
            tol[rows] += 2.0 ** -24 * ((self.K + self.rank + 2) * abs(s) * (mag_u @ b.abs().t()) + (self.rank + 2) * self.r[rows, :self.N].to(F64).abs())
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
        err = (got - want).abs()
        assert (err <= tol).all(), f"worst {(err / tol).max()} of the bound"
        assert torch.isnan(out[self.live:]).all() or out is self.keep[0]["r"], "rows behind the last sequence were written"
        if out is not self.keep[0]["r"]:
            assert torch.isnan(out[:, self.N:]).all(), "columns behind the last feature were written"


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 96, 128])
@pytest.mark.parametrize("lens,adapters", [
    ([1], [0]), ([1, 1, 1, 1], [2, -1, 0, 2]), ([0, 7, 0, 16, 17], [0, 1, -1, 2, 0]), ([40, 1, 30], [1, 7, 0]), ([130, 65, 64], [2, 0, -5])])
@pytest.mark.parametrize("K,N", [(64, 8), (256, 264), (1088, 512)])
def test_lora(lens, adapters, K, N, rank):
    c = Case(lens, adapters, K, N, rank, seed=rank + len(lens), pad=8)
    c.check(c.call())
    c.check(c.call(in_place=True))


def test_lora_without_scale_and_with_one_adapter():
    c = Case([3, 90], [0, 0], 512, 1056, 16, n=1, scale=False)
    c.check(c.call())


def test_lora_long_k_and_many_sequences():
    """K in ranges over workgroups; more sequences than one step of the search covers, some without a row."""
    c = Case([1, 2], [1, 0], 6144, 136, 64)
    assert _lib.load().coda_lora_workspace_bytes(c.T, c.B, c.N, c.K, c.rank) > c.T * c.rank * 4
    c.check(c.call())
    for B in (200, 600):
        lens = [(i * 5) % 4 for i in range(B)]
        for rank in (16, 40):                               # one launch, two launches
            c = Case(lens, [(i * 3) % 5 - 1 for i in range(B)], 128, 72, rank, n=3)
            c.check(c.call())


def test_lora_nothing_leaks_between_rows():
    """A row of infinities poisons itself alone, also inside a tile; a sequence without an adapter never sees X."""
    c = Case([20, 5, 33], [0, -1, 2], 256, 264, 32, seed=9)
    want = c.call().clone()
    d = c.device()
    d["x"][7] = float("inf")
    d["x"][20:25] = float("nan")
    out = c.call(d)
    others = [r for r in range(c.live) if r != 7]
    assert torch.equal(out[others], want[others]) and not torch.isfinite(out[7, :264]).any()


def test_lora_same_bits_streams_and_graph():
    c = Case([1, 40, 3], [2, 0, 1], 2048, 512, 16, seed=4)
    want = c.call().clone()
    d, ws = c.keep
    assert torch.equal(c.call()[:c.live], want[:c.live])
    out = torch.full_like(want, float("nan"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.call(d, out=out, ws=ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(out[:c.live], want[:c.live])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.call(d, out=out, ws=ws)
    for turn in range(3):
        c.adapter = (c.adapter + 1) % 3                     # read when the graph runs
        d["adapter"].copy_(c.adapter)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got[:c.live], c.call()[:c.live])
        c.check(got)


@pytest.mark.parametrize("rank", [8, 16, 24, 32])
@pytest.mark.parametrize("K,N", [(64, 1032), (1984, 264), (2048, 4096), (8192, 72)])
def test_lora_one_launch(K, N, rank):
    """Short sequences, small adapters: the single launch (no workspace), against the same bound; 33 sequences so that some tiles are
    alone on their CU and some are not."""
    lens = [(i * 5) % 4 for i in range(33)]
    lens[7] = 21                                             # two tiles
    c = Case(lens, [(i * 3) % 5 - 1 for i in range(33)], K, N, rank, seed=rank, pad=8)
    assert (_lib.load().coda_lora_workspace_bytes(c.T, c.B, N, K, rank) == 0) == (rank * K <= 65536)
    c.check(c.call())
    c.check(c.call(in_place=True))


@pytest.mark.parametrize("rank", [16, 64])
@pytest.mark.parametrize("starts", [[0, 90, 40, 60], [-7, 20, 200, 30], [300, 300, 300, 300]])
def test_lora_starts_that_make_no_sense(starts, rank):
    """Starts that decrease or leave [0, T]: rows come out wrong or not at all, and nothing else is touched."""
    c = Case([30, 30, 30], [0, 1, 2], 128, 72, rank)
    c.seq_start = torch.tensor(starts, dtype=torch.int32)
    guard = torch.full((c.T + 64, 72), 7.0, device=DEV, dtype=BF)
    c.call(out=guard[32:32 + c.T])
    torch.cuda.synchronize()
    assert (guard[:32] == 7).all() and (guard[32 + c.T:] == 7).all()


@pytest.mark.parametrize("rank", [16, 24, 64])
def test_lora_infinities_and_the_end_of_the_range(rank):
    """An infinity in X comes out as the infinity that the formula gives, not as a NaN; products X A^T between bf16's largest value and fp32's
    are kept.  One launch (ranks 16, 24) and two."""
    c = Case([3, 4, 2], [0, 1, -1], 256, 264, rank, n=2, scale=False)
    assert (_lib.load().coda_lora_workspace_bytes(c.T, c.B, c.N, c.K, rank) == 0) == (rank < 64)
    c.a[0], c.b[0] = c.a[0].abs() + 2.0 ** -6, c.b[0].abs() + 2.0 ** -6       # no zeros: 0 * inf would be a NaN by right
    c.x[0, 5], c.x[1, 9] = float("inf"), float("-inf")
    c.a[1], c.b[1] = 0, 0
    c.a[1, 3, :2], c.b[1, :, 3] = 1, 2.0 ** -10                # U[3] = x0 + x1, all else 0
    c.x[3, :2] = torch.tensor([3.3895313892515355e38, 1e36])   # bf16's largest value, and beyond half a step of it
    c.x[4, :2] = -c.x[3, :2]
    out = c.call()
    torch.cuda.synchronize()
    assert (out[0, :c.N] == float("inf")).all() and (out[1, :c.N] == float("-inf")).all()
    out[0, :c.N], out[1, :c.N] = c.r[0, :c.N].to(DEV), c.r[1, :c.N].to(DEV)
    c.x[0], c.x[1] = 0, 0
    c.check(out)


def plan(c):
    """(16-token blocks a tile, K ranges, elements of a range, features of a workgroup) of a call in two launches, as lora.hip cuts it."""
    cus, up = torch.cuda.get_device_properties(0).multi_processor_count, lambda a, b: -(-a // b)
    mt = 1 if c.T / c.B <= 16 else 2
    tiles = max(up(c.T, 16 * mt), c.B)
    nslice = 512 if tiles * up(c.N, 512) >= cus else 256
    most = (2 * c.K + 4 * c.N) // 8 // (4 * c.rank * (1 + up(c.N, nslice)))
    ks = max(1, min(max(min(up(4 * cus, tiles), most), up(cus, tiles)), c.K // 256))
    chunk = up(up(c.K, ks), 64) * 64
    split = up(c.K, chunk)
    bytes_ = _lib.load().coda_lora_workspace_bytes(c.T, c.B, c.N, c.K, c.rank)
    assert bytes_ == (c.T // (16 * mt) + c.B) * 16 + split * c.T * c.rank * 4
    return mt, split, chunk, nslice


def both_places(c):
    c.check(c.call())
    out = c.call(in_place=True)
    c.check(out)
    assert torch.equal(out[c.live:].cpu(), c.r[c.live:]) and torch.equal(out[:, c.N:].cpu(), c.r[:, c.N:])


@pytest.mark.parametrize("rank", [32, 64, 128])
@pytest.mark.parametrize("K,N", [(1088, 520), (2048, 1056)])
@pytest.mark.parametrize("most", [16, 40])
def test_lora_several_steps_of_both_products(most, K, N, rank):
    """Many tiles: a workgroup of the first launch takes more than two steps of 256 elements of K, one of the second more than one step of
    256 features, the last of them short; also where it only copies."""
    lens = [1 + (i * 7) % 16 if most == 16 else 17 + (i * 7) % 24 for i in range(300)]
    c = Case(lens, [(i * 3) % 5 - 1 for i in range(300)], K, N, rank, seed=rank, pad=8, spare=3)
    mt, split, chunk, nslice = plan(c)
    assert mt == (1 if most == 16 else 2) and chunk > 512 and nslice == 512
    both_places(c)


def test_lora_blocks_over_ranges_of_several_steps():
    """32 blocks of 32 tokens, K 6144 in eight ranges of three steps each."""
    c = Case([32] * 32, [(i * 3) % 9 - 1 for i in range(32)], 6144, 2048, 64, n=8, seed=3, pad=8)
    assert plan(c) == (2, 8, 768, 256)
    both_places(c)
