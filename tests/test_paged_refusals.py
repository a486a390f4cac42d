"""Argument checks of the ragged-batch entry points (paged cache, low-rank adapters): every refusal returns its code and
words before anything is launched, so none of this needs a GPU - and none of these calls may reach one."""
import os

import pytest
import torch

from coda_amd import _lib

P = 1 << 20          # stands for an aligned device pointer: a refused call never follows it


@pytest.fixture(scope="module", autouse=True)
def _built():
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()


APPEND = dict(qkv=P, ld_qkv=32 * 128, q_out=P, ld_q=16 * 128, q_weight=P, k_weight=P, cos=P, sin=P, max_pos=64, seq_start=P, pos0=P, B=2,
              T=4, page_table=P, ld_table=8, max_pages=8, k_cache=P, v_cache=P, page_stride=8 * 16 * 128, num_pages=16, page_size=16,
              cache_type=0, k_scale=1.0, v_scale=1.0, n_q=16, n_kv=8, eps=1e-6, flags=0, stream=None)
ATTN = dict(q=P, ld_q=16 * 128, out=P, ld_out=16 * 128, seq_start=P, pos0=P, kv_len=P, B=2, T=4, page_table=P, ld_table=8, max_pages=8,
            k_cache=P, v_cache=P, page_stride=8 * 16 * 128, num_pages=16, page_size=16, cache_type=0, k_scale=1.0, v_scale=1.0,
            max_kv=128, n_q=16, n_kv=8, scale=0.1, mask_block=0, workspace=P, workspace_bytes=1 << 30, stream=None)

NAN, INF = float("nan"), float("inf")
PAGES = [  # the checks of a cache are the same for both entry points
    (dict(k_cache=None), "ARG", "null cache"), (dict(v_cache=None), "ARG", "null cache"), (dict(page_table=None), "ARG", "null cache"),
    (dict(cache_type=2), "ARG", "cache type"), (dict(cache_type=-1), "ARG", "cache type"),
    (dict(cache_type=1, k_scale=0.0), "ARG", "scales"), (dict(cache_type=1, v_scale=-1.0), "ARG", "scales"),
    (dict(cache_type=1, v_scale=NAN), "ARG", "scales"), (dict(cache_type=1, k_scale=INF), "ARG", "scales"),
    (dict(cache_type=1, k_scale=1e-38), "ARG", "scales"),
    (dict(num_pages=0), "SHAPE", "page table"), (dict(page_size=0), "SHAPE", ""), (dict(page_size=-16), "SHAPE", ""),
    (dict(ld_table=7), "SHAPE", "page table"), (dict(max_pages=1 << 28, ld_table=1 << 28), "SHAPE", "2^31"),
    (dict(page_stride=8 * 16 * 128 - 8), "SHAPE", "page_stride"), (dict(page_stride=8 * 16 * 128 + 4), "ALIGN", "16 bytes"),
    (dict(k_cache=P + 8), "ALIGN", "16 bytes"), (dict(v_cache=P + 2), "ALIGN", "16 bytes"),
    (dict(cache_type=1, page_stride=8 * 16 * 128 + 8), "ALIGN", "16 bytes"),
]
BATCH = [(dict(B=0), "SHAPE", ""), (dict(B=-1), "SHAPE", ""), (dict(T=0), "SHAPE", ""), (dict(n_q=0), "SHAPE", ""), (dict(n_kv=0), "SHAPE", ""),
         (dict(seq_start=None), "ARG", "null"), (dict(pos0=None), "ARG", "null")]


def refused(name, base, change, code, words):
    args = {**base, **change}
    with pytest.raises(_lib.CodaHipError) as e:
        _lib.call(name, *args.values())
    assert f"CODA_ERR_{code}" in str(e.value), str(e.value)
    assert words in str(e.value)
    # worded, and by its own name: a stale message of another call would not be shown
    assert f" {name}: " in str(e.value), str(e.value)


@pytest.mark.parametrize("change,code,words", PAGES + BATCH + [
    (dict(max_pos=0), "SHAPE", ""), (dict(ld_qkv=32 * 128 - 8), "SHAPE", "stride"), (dict(ld_q=16 * 128 - 8), "SHAPE", "stride"),
    (dict(qkv=None), "ARG", "null"), (dict(q_out=None), "ARG", "null"), (dict(cos=None), "ARG", "null"), (dict(sin=None), "ARG", "null"),
    (dict(q_weight=None), "ARG", "together"), (dict(k_weight=None), "ARG", "together"), (dict(flags=2), "ARG", "flag"),
    (dict(qkv=P + 2), "ALIGN", "16 bytes"), (dict(cos=P + 8), "ALIGN", "16 bytes"), (dict(k_weight=P + 4), "ALIGN", "16 bytes"),
    (dict(ld_qkv=32 * 128 + 4), "ALIGN", "16 bytes"), (dict(ld_q=16 * 128 + 2), "ALIGN", "16 bytes"),
    (dict(n_q=2000000, ld_qkv=1 << 40), "SHAPE", "heads"),
])
def test_append_refuses(change, code, words):
    refused("coda_paged_append", APPEND, change, code, words)


@pytest.mark.parametrize("change,code,words", PAGES + BATCH + [
    (dict(kv_len=None), "ARG", "null"), (dict(q=None), "ARG", "null"), (dict(out=None), "ARG", "null"),
    (dict(n_q=15), "SHAPE", "n_q"), (dict(max_kv=129), "SHAPE", "max_kv"), (dict(max_kv=-1), "SHAPE", "max_kv"),
    (dict(max_pages=0), "SHAPE", ""), (dict(ld_q=16 * 128 - 8), "SHAPE", "stride"), (dict(ld_out=16 * 128 - 8), "SHAPE", "stride"),
    (dict(scale=0.0), "ARG", "scale"), (dict(scale=-0.1), "ARG", "scale"), (dict(scale=NAN), "ARG", "scale"), (dict(scale=INF), "ARG", "scale"),
    (dict(scale=1e-31), "ARG", "scale"), (dict(scale=1e20, cache_type=1, k_scale=1e20), "ARG", "k_scale"),
    (dict(max_kv=(1 << 30) + 1, max_pages=1 << 27, ld_table=1 << 27), "SHAPE", "max_kv"),
    (dict(mask_block=-1), "ARG", "mask_block"), (dict(q=P + 8), "ALIGN", ""), (dict(ld_out=16 * 128 + 4), "ALIGN", ""),
    (dict(T=1 << 28), "SHAPE", "2^31"), (dict(T=(1 << 27) + 1, n_q=8, n_kv=4), "SHAPE", "2^28"),
    # 4096 keys are more than one range: the workspace has to be there
    (dict(max_kv=4096, max_pages=256, ld_table=256, workspace_bytes=1024), "ARG", "workspace"),
    (dict(max_kv=4096, max_pages=256, ld_table=256, workspace=None), "ARG", "workspace"),
    (dict(max_kv=4096, max_pages=256, ld_table=256, workspace=P + 4), "ALIGN", "workspace"),
])
def test_attn_refuses(change, code, words):
    refused("coda_paged_attn", ATTN, change, code, words)


@pytest.mark.skipif(torch.cuda.is_available(), reason="what a machine without a GPU answers")
def test_no_device_is_said_and_not_an_older_error():
    refused("coda_paged_append", APPEND, dict(flags=2), "ARG", "flag")
    with pytest.raises(_lib.CodaHipError) as e:
        _lib.call("coda_paged_attn", *ATTN.values())
    assert "CODA_ERR_LAUNCH hipGetDevice: " in str(e.value), str(e.value)


def test_attn_workspace_sizes():
    size = _lib.load().coda_paged_attn_workspace_bytes
    assert size(1, 1, 0, 16, 8) == 0 and size(1, 1, 256, 16, 8) == 0          # one range of keys: joined by nobody
    assert size(1, 1, 4096, 16, 8) > 0
    assert size(0, 1, 4096, 16, 8) == 0 and size(1, 1, 4096, 16, 7) == 0      # sizes that the call itself refuses
    for T, B, kv in ((1, 1, 40960), (4, 4, 40960), (128, 128, 2048), (1024, 32, 384), (8192, 8, 4096)):
        # a head, and a partial output and two numbers per range, token and head; no ranges under 128 keys, nor over 64 MiB of them
        n = size(T, B, kv, 16, 8)
        assert n == 0 or (n - 256) % (T * 16 * 130 * 4) == 0 and n - 256 <= min(kv // 128 * T * 16 * 130 * 4, 64 << 20)


@pytest.mark.parametrize("name,change,code,words", [
    # n_kv * page_size * 128 is 2^64: a page_stride of any length would pass for a page
    ("coda_paged_attn", dict(T=1, n_q=1 << 30, n_kv=1 << 30, ld_q=1 << 38, ld_out=1 << 38, page_size=1 << 27, page_stride=2048), "SHAPE", "heads"),
    ("coda_paged_attn", dict(T=1, n_q=(1 << 20) + 1, n_kv=(1 << 20) + 1, ld_q=1 << 38, ld_out=1 << 38, page_stride=1 << 40), "SHAPE", "heads"),
    # the search for a token's sequence takes (B + 63) / 64 of them a step
    ("coda_paged_append", dict(B=(1 << 31) - 1), "SHAPE", "2^30"), ("coda_paged_append", dict(B=(1 << 30) + 1), "SHAPE", "2^30"),
    ("coda_lora_bf16", dict(N=2147483640, ldr=1 << 31, ldc=1 << 31), "SHAPE", "2^30"),
    ("coda_lora_bf16", dict(K=2147483584, ldx=1 << 31), "SHAPE", "2^30"),
])
def test_sizes_whose_sums_would_wrap(name, change, code, words):
    refused(name, {"coda_paged_append": APPEND, "coda_paged_attn": ATTN, "coda_lora_bf16": LORA}[name], change, code, words)


def test_workspaces_of_sizes_that_would_wrap():
    lib, big = _lib.load(), (1 << 31) - 1
    assert lib.coda_paged_attn_workspace_bytes(big, big, big, big, 1) == 0 and lib.coda_paged_attn_workspace_bytes(1 << 30, 1, 1 << 30, 8, 8) == 0
    assert lib.coda_lora_workspace_bytes(4, 2, big, 64, 8) == 0 and lib.coda_lora_workspace_bytes(4, 2, 64, big, 8) == 0
    assert lib.coda_lora_workspace_bytes(big, 2, 64, 64, 8) == 0 and lib.coda_lora_workspace_bytes(4, 2, 64, 64, big) == 0


LORA = dict(X=P, ldx=256, A=P, Bw=P, scale=None, seq_start=P, adapter=P, B=2, T=4, n_adapters=3, rank=64, R=P, ldr=512, C=P, ldc=512, N=512,
            K=256, workspace=P, workspace_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("name,change,words", [
    ("coda_paged_append", dict(T=(1 << 26) + 1, n_q=1, n_kv=1), "too many rows"),                    # four tokens a workgroup of 256
    ("coda_paged_attn", dict(T=1 << 24, B=1 << 24, n_q=1, n_kv=1), "too many tiles"),                # 2^24 sequences of a token
    ("coda_paged_attn", dict(T=3200, B=1 << 22, n_q=8), "too many tiles"),                            # almost all sequences empty
    ("coda_lora_bf16", dict(T=1 << 24, B=1 << 24, workspace_bytes=1 << 40), "too many tiles"),
])
def test_launches_of_too_many_work_items(name, change, words):
    """2^32 work items and more are no launch; fewer than 2^31 workgroups all the same."""
    refused(name, {"coda_paged_append": APPEND, "coda_paged_attn": ATTN, "coda_lora_bf16": LORA}[name], change, "SHAPE", words)


@pytest.mark.parametrize("change,code,words", [
    (dict(B=0), "SHAPE", "positive"), (dict(T=0), "SHAPE", "positive"), (dict(T=-3), "SHAPE", "positive"), (dict(n_adapters=0), "SHAPE", "positive"),
    (dict(T=(1 << 28) + 1), "SHAPE", "2^28"), (dict(N=0), "SHAPE", "positive"), (dict(K=0), "SHAPE", "positive"), (dict(rank=0), "SHAPE", "rank"), (dict(rank=12), "SHAPE", "rank"),
    (dict(rank=136), "SHAPE", "rank"), (dict(K=224), "SHAPE", "K % 64"), (dict(N=508), "SHAPE", "N % 8"), (dict(ldx=248), "SHAPE", "stride"),
    (dict(ldr=504), "SHAPE", "stride"), (dict(ldc=504), "SHAPE", "stride"),
    *[(dict([(n, None)]), "ARG", "null") for n in ("X", "A", "Bw", "seq_start", "adapter", "R", "C")],
    *[(dict([(n, P + 8)]), "ALIGN", "16 bytes") for n in ("X", "A", "Bw", "R", "C")],
    (dict(ldx=260), "ALIGN", "16 bytes"), (dict(ldr=516), "ALIGN", "16 bytes"), (dict(ldc=516), "ALIGN", "16 bytes"),
    (dict(workspace=None), "ARG", "workspace"), (dict(workspace_bytes=64), "ARG", "workspace"), (dict(workspace=P + 8), "ALIGN", "workspace"),
])
def test_lora_refuses(change, code, words):
    refused("coda_lora_bf16", LORA, change, code, words)


def test_lora_workspace_sizes():
    size = _lib.load().coda_lora_workspace_bytes
    assert size(0, 1, 512, 256, 16) == 0 and size(4, 2, 512, 256, 0) == 0
    assert size(32, 32, 4096, 2048, 16) == 0                                  # single tokens, small adapters: one launch, no slabs
    for T, B, K, rank in ((1, 1, 6144, 16), (32, 32, 2048, 64), (1024, 32, 6144, 64), (16384, 32, 2048, 128)):
        # 16 bytes a tile (at most T / 16 + B of them), and U in at most K / 256 slabs of fp32
        n = size(T, B, 2048, K, rank)
        assert T * rank * 4 < n <= (T // 16 + B) * 16 + K // 256 * T * rank * 4
