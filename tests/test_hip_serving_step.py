"""The ragged-batch operators together, as a serving step uses them: projection + adapters, append, attention, for every layer
of a small decoder whose other products are the library's own."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from coda_amd import CoDAConfig, _lib  # noqa: E402
from coda_amd.engine import HipEngine  # noqa: E402

DEV = "cuda"
BF = torch.bfloat16
N_Q, N_KV, D, H, I, LAYERS, V = 4, 2, 128, 256, 512, 3, 512
QKV = (N_Q + 2 * N_KV) * D


def _s():
    return torch.cuda.current_stream().cuda_stream


@pytest.fixture(scope="module")
def engine():
    from oracle import ref_cpu
    d = ref_cpu.Dims(vocab=V, hidden=H, inter=I, heads=N_Q, kv_heads=N_KV, head_dim=D, layers=LAYERS, mask_id=V - 1, pad_id=500,
                     max_pos=1024)
    sd = {k: v.to(BF) for k, v in ref_cpu.make_state_dict(d, 7, lm_head_gain=8.0, norm_jitter=0.1).items()}
    cfg = CoDAConfig(vocab_size=V, hidden_size=H, intermediate_size=I, num_attention_heads=N_Q, num_key_value_heads=N_KV, head_dim=D,
                     num_hidden_layers=LAYERS)
    return HipEngine(cfg, sd, torch.device("cuda:0"))


class Server:
    """Caches of every layer, one page table; step() runs new tokens of some sequences through the decoder."""

    def __init__(self, eng, B, max_len, page, adapters=None, cache=_lib.CACHE_BF16, flags=_lib.APPEND_STEPWISE):
        self.eng, self.B, self.page, self.cache, self.flags = eng, B, page, cache, flags
        self.max_pages = -(-max_len // page)
        g = torch.Generator().manual_seed(3)
        self.num_pages = B * self.max_pages
        self.table = torch.randperm(self.num_pages, generator=g).view(B, self.max_pages).to(torch.int32).to(DEV)
        dtype = torch.float8_e4m3fn if cache == _lib.CACHE_E4M3 else BF
        shape = (LAYERS, self.num_pages, N_KV, page, D)
        self.k, self.v = (torch.full(shape, float("nan"), dtype=torch.float32).to(dtype).to(DEV) for _ in range(2))
        self.length = [0] * B
        inv = 1.0 / (eng.theta ** (torch.arange(0, D, 2, dtype=torch.int64).float() / D))
        ang = torch.arange(max_len).float()[:, None] * inv[None, :]
        ang = torch.cat((ang, ang), -1)
        self.cos, self.sin = ang.cos().to(BF).to(DEV), ang.sin().to(BF).to(DEV)
        self.adapters = adapters

    def step(self, ids, mask, rewind=0, keep=False):
        """ids: new token ids per sequence (lists, may be empty); `rewind`: positions of each sequence that are written anew; `keep`: what
        lies behind the new tokens stays part of its sequence."""
        e, s = self.eng, _s()
        lens = [len(x) for x in ids]
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        T = starts[-1]
        past = [n - rewind for n in self.length]
        self.length = [max(p + n, old) if keep else p + n for p, n, old in zip(past, lens, self.length)]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
        seq, pos0, kv = i32(starts), i32(past), i32(self.length)
        flat = torch.tensor([t for x in ids for t in x], dtype=torch.int64, device=DEV)
        new = lambda *shape: torch.empty(*shape, dtype=BF, device=DEV)
        h, a, qkv, q, ao, mlp = new(T, H), new(T, H), new(T, QKV), new(T, N_Q * D), new(T, N_Q * D), new(T, I)
        keep = [seq, pos0, kv, flat, h, a, qkv, q, ao, mlp]
        _lib.call("coda_embed_gather", flat.data_ptr(), e.embed.data_ptr(), h.data_ptr(), T, V, H, s)
        lib, max_kv = _lib.load(), max(self.length)
        ws = torch.empty(max(16, lib.coda_paged_attn_workspace_bytes(T, self.B, max_kv, N_Q, N_KV)), dtype=torch.uint8, device=DEV)

        def gemm(x, w, out, epi, r=None):
            _lib.call("coda_gemm_bf16", x.data_ptr(), x.stride(0), None, w.data_ptr(), w.stride(0), out.data_ptr(), out.stride(0),
                      None if r is None else r.data_ptr(), 0 if r is None else r.stride(0), T, w.shape[0], w.shape[1], epi, s)

        def norm(x, w, out):
            _lib.call("coda_rmsnorm", x.data_ptr(), x.stride(0), w.data_ptr(), out.data_ptr(), out.stride(0), T, H, e.eps, s)

        for li, lw in enumerate(e.lw):
            norm(h, lw["n_in"], a)
            gemm(a, lw["wqkv"], qkv, _lib.EPI_PLAIN)
            if self.adapters:
                la, lb, which = self.adapters[li]
                n, r, _ = la.shape
                size = lib.coda_lora_workspace_bytes(T, self.B, QKV, H, r)
                lws = torch.empty(max(16, size), dtype=torch.uint8, device=DEV)
                keep.append(lws)
                _lib.call("coda_lora_bf16", a.data_ptr(), H, la.data_ptr(), lb.data_ptr(), None, seq.data_ptr(), which.data_ptr(), self.B, T, n,
                          r, qkv.data_ptr(), QKV, qkv.data_ptr(), QKV, QKV, H, lws.data_ptr(), size, s)
            geo = (self.table.data_ptr(), self.max_pages, self.max_pages, self.k[li].data_ptr(), self.v[li].data_ptr(),
                   N_KV * self.page * D, self.num_pages, self.page, self.cache, 1 / 32, 1 / 64)
            _lib.call("coda_paged_append", qkv.data_ptr(), QKV, q.data_ptr(), N_Q * D, lw["qn"].data_ptr(), lw["kn"].data_ptr(),
                      self.cos.data_ptr(), self.sin.data_ptr(), self.cos.shape[0], seq.data_ptr(), pos0.data_ptr(), self.B, T, *geo, N_Q,
                      N_KV, e.eps, self.flags, s)
            _lib.call("coda_paged_attn", q.data_ptr(), N_Q * D, ao.data_ptr(), N_Q * D, seq.data_ptr(), pos0.data_ptr(), kv.data_ptr(),
                      self.B, T, *geo, max_kv, N_Q, N_KV, 1 / math.sqrt(D), mask, ws.data_ptr(), ws.numel(), s)
            gemm(ao, lw["wo"], h, _lib.EPI_RESIDUAL, r=h)
            norm(h, lw["n_post"], a)
            gemm(a, lw["wgu"], mlp, _lib.EPI_SWIGLU)
            gemm(mlp, lw["wd"], h, _lib.EPI_RESIDUAL, r=h)
        out = new(T, H)
        norm(h, e.final_norm, out)
        torch.cuda.synchronize()
        del keep
        return out, starts


def rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


# one bf16 rounding per layer and branch that falls the other way moves the result by about 2^-8 of it; three layers of two branches
BAND = 6 * 2.0 ** -8


def test_whole_prompts_equal_the_uncached_forward(engine):
    """Every position appended and attended at once, unmasked: the uncached bidirectional forward."""
    g = torch.Generator().manual_seed(1)
    B, L = 3, 70
    ids = torch.randint(0, V - 2, (B, L), generator=g)
    want = engine.forward_hidden(ids.to(DEV)).clone()
    out, _ = Server(engine, B, L, 16).step(ids.tolist(), 0)
    assert rel(out, want) < BAND


def test_denoise_block_over_kept_keys(engine):
    """A block in the middle of the sequence is run again over the kept keys and values of the same state: the same hidden rows."""
    g = torch.Generator().manual_seed(2)
    B, L, lo, n = 2, 96, 64, 32
    ids = torch.randint(0, V - 2, (B, L), generator=g).tolist()
    srv = Server(engine, B, L, 32)
    whole, _ = srv.step(ids, 0)
    again, _ = srv.step([x[lo:lo + n] for x in ids], 0, rewind=L - lo)
    assert rel(again.view(B, n, H), whole.view(B, L, H)[:, lo:lo + n]) < BAND


@pytest.mark.parametrize("page", [16, 7])
def test_denoise_block_with_keys_on_both_sides(engine, page):
    """A block in the middle, later positions kept: unmasked, the hidden rows of the whole sequence; in blocks of 32, those of the block-causal
    whole, whatever lies behind."""
    g = torch.Generator().manual_seed(5)
    B, L, lo, n = 2, 96, 32, 32
    ids = torch.randint(0, V - 2, (B, L), generator=g).tolist()
    block = [x[lo:lo + n] for x in ids]
    for mask in (0, 32):
        srv = Server(engine, B, L, page)
        whole, _ = srv.step(ids, mask)
        again, _ = srv.step(block, mask, rewind=L - lo, keep=True)
        assert srv.length == [L] * B
        assert rel(again.view(B, n, H), whole.view(B, L, H)[:, lo:lo + n]) < BAND
        short, _ = srv.step(block, mask, rewind=L - lo)          # the same without them
        if mask:
            assert rel(short, again) < BAND
        else:
            assert rel(short, again) > BAND


@pytest.mark.parametrize("page,cache", [(16, _lib.CACHE_BF16), (7, _lib.CACHE_BF16), (64, _lib.CACHE_E4M3)])
@pytest.mark.parametrize("adapted", [False, True])
def test_ragged_chunks_equal_whole_prompts(engine, page, cache, adapted):
    """Causal: requests of different lengths in ragged chunks - prompts, blocks, single tokens, requests that sit a step out - give
    the hidden rows that whole prompts give, each with its own adapter."""
    g = torch.Generator().manual_seed(4)
    lens = [90, 41, 133, 1]
    ids = [torch.randint(0, V - 2, (n,), generator=g).tolist() for n in lens]
    adapters = None
    if adapted:
        which = torch.tensor([1, -1, 0, 1], dtype=torch.int32, device=DEV)
        adapters = [((torch.randn(2, 16, H, generator=g) * H ** -0.5).to(BF).to(DEV), (torch.randn(2, QKV, 16, generator=g) * 0.25).to(BF).to(DEV),
                     which) for _ in range(LAYERS)]
    whole, starts = Server(engine, 4, 133, page, adapters, cache, 0).step(ids, 1)
    if adapted:
        plain, _ = Server(engine, 4, 133, page, None, cache, 0).step(ids, 1)
        second = slice(starts[1], starts[2])                # the request without an adapter
        assert torch.equal(plain[second], whole[second]) and rel(plain, whole) > BAND
    srv = Server(engine, 4, 133, page, adapters, cache, 0)
    cuts = [[0, 50, 50, 82, 89, 90], [0, 0, 40, 41, 41, 41], [0, 1, 33, 130, 132, 133], [0, 0, 0, 0, 0, 1]]
    got = [[] for _ in ids]
    for i in range(5):
        out, st = srv.step([x[c[i]:c[i + 1]] for x, c in zip(ids, cuts)], 1)
        for b in range(4):
            got[b].append(out[st[b]:st[b + 1]])
    for b in range(4):
        # e4m3: a key that rounds the other way moves by a step of 2^-3, some of the time; averaged over the keys of a row
        assert rel(torch.cat(got[b]), whole[starts[b]:starts[b + 1]]) < (BAND if cache == _lib.CACHE_BF16 else 4 * BAND)


def test_captured_step_replayed_over_growing_caches():
    """Projection, adapters, append and attention of single tokens as one captured graph: replayed while the lengths on the device grow,
    with eager work between the replays, against the same calls made one by one on their own caches."""
    g = torch.Generator().manual_seed(6)
    B, page, max_kv, rank, n_ad = 5, 16, 3000, 64, 3
    max_pages = -(-max_kv // page)
    rnd = lambda *shape, scale=1.0: (torch.randn(*shape, generator=g) * scale).to(BF).to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    w, la, lb = rnd(QKV, H, scale=H ** -0.5), rnd(n_ad, rank, H, scale=H ** -0.5), rnd(n_ad, QKV, rank, scale=0.1)
    qn, kn = rnd(D), rnd(D)
    ang = torch.arange(max_kv)[:, None] / 1e6 ** (torch.arange(0, D, 2) / D)[None, :]
    cos, sin = (f(torch.cat((ang, ang), -1)).to(BF).to(DEV) for f in (torch.cos, torch.sin))
    table = torch.randperm(B * max_pages, generator=g).view(B, max_pages).to(torch.int32).to(DEV)
    k0, v0 = rnd(B * max_pages, N_KV, page, D), rnd(B * max_pages, N_KV, page, D)
    seq, pos0, kv, which = i32(list(range(B + 1))), i32([2900, 0, 15, 1000, 2047]), i32([0] * B), i32([0, 2, -1, 1, 0])
    x = rnd(B, H)
    lib = _lib.load()

    class Side:
        def __init__(self):
            self.k, self.v = k0.clone(), v0.clone()
            self.qkv, self.out = torch.empty(B, QKV, dtype=BF, device=DEV), torch.empty(B, N_Q * D, dtype=BF, device=DEV)
            sizes = lib.coda_lora_workspace_bytes(B, B, QKV, H, rank), lib.coda_paged_attn_workspace_bytes(B, B, max_kv, N_Q, N_KV)
            assert min(sizes) > 0                               # two launches each
            self.ws = [torch.empty(n, dtype=torch.uint8, device=DEV) for n in sizes]

        def enqueue(self):
            s, qkv = _s(), self.qkv
            _lib.call("coda_gemm_bf16", x.data_ptr(), H, None, w.data_ptr(), H, qkv.data_ptr(), QKV, None, 0, B, QKV, H, _lib.EPI_PLAIN, s)
            _lib.call("coda_lora_bf16", x.data_ptr(), H, la.data_ptr(), lb.data_ptr(), None, seq.data_ptr(), which.data_ptr(), B, B, n_ad, rank,
                      qkv.data_ptr(), QKV, qkv.data_ptr(), QKV, QKV, H, self.ws[0].data_ptr(), self.ws[0].numel(), s)
            geo = (table.data_ptr(), max_pages, max_pages, self.k.data_ptr(), self.v.data_ptr(), N_KV * page * D, B * max_pages, page,
                   _lib.CACHE_BF16, 1.0, 1.0)
            _lib.call("coda_paged_append", qkv.data_ptr(), QKV, qkv.data_ptr(), QKV, qn.data_ptr(), kn.data_ptr(), cos.data_ptr(),
                      sin.data_ptr(), max_kv, seq.data_ptr(), pos0.data_ptr(), B, B, *geo, N_Q, N_KV, 1e-6, 0, s)
            _lib.call("coda_paged_attn", qkv.data_ptr(), QKV, self.out.data_ptr(), N_Q * D, seq.data_ptr(), pos0.data_ptr(), kv.data_ptr(), B, B,
                      *geo, max_kv, N_Q, N_KV, 1 / math.sqrt(D), 1, self.ws[1].data_ptr(), self.ws[1].numel(), s)

    kv.copy_(pos0 + 1)
    eager, captured = Side(), Side()
    captured.enqueue()                                          # first launches outside the capture; its caches are made anew
    torch.cuda.synchronize()
    captured.k.copy_(k0)
    captured.v.copy_(v0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.enqueue()
    for turn in range(4):
        x.copy_(rnd(B, H))
        kv.copy_(pos0 + 1)
        graph.replay()
        eager.enqueue()
        torch.cuda.synchronize()
        assert torch.isfinite(eager.out).all()
        for a, b in ((captured.out, eager.out), (captured.k, eager.k), (captured.v, eager.v)):
            assert torch.equal(a, b), turn
        pos0 += 7                                               # also leaves slots that nobody wrote: those of the random cache
