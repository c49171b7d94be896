"""Addresses off the boundary that a kernel's loads and stores need are refused before any launch (C, without a device): results
that are written two bf16 at a time, caches that are read four or sixteen bytes at a time."""
import pytest

from test_kv8_refusals import ALIGN, FEW, ROWS, TC, TILES, _entry, some


@pytest.mark.parametrize("change", [dict(), dict(ws=some, n_ctas=1, n_splits=0)], ids=["clusters", "dealt out"])
@pytest.mark.parametrize("off", [2, 6])
def test_results_of_single_tokens_off_a_pair(change, off):
    f = _entry("attention_kv8@hd64", "plm_kv8_attention_few", ["-DPLM_HD=64"])
    assert FEW.call(f, **{**change, "out": some + off}) == ALIGN


def test_results_of_prompts_off_a_pair():
    assert TILES.call(_entry("attention_kv8@hd80", "plm_kv8_attention_tiles", ["-DPLM_HD=80"]), out=some + 2) == ALIGN
    assert TC.call(_entry("attention_kv8_tc@hd64", "plm_kv8_attention_tc", ["-DPLM_HD=64"]), out=some + 2) == ALIGN


@pytest.mark.parametrize("name", ["kc", "vc"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_caches_off_four_bytes(name, off):
    assert ROWS.call(_entry("kv8", "plm_kv8_attention_rows"), **{name: some + off}) == ALIGN


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 80])
def test_faces_refuse_views_off_the_boundary(hd):
    import torch
    from picolm_b200 import ops
    from test_kv8_refusals import _tensors

    def off(t, n=1):                                                  # the same contents, n elements behind a boundary
        flat = torch.zeros(t.numel() + n, dtype=t.dtype, device=t.device)
        return flat[n:].view(t.shape)

    for name in ("attention_kv8_decode", "attention_kv8_prefill"):
        for dtype, wrong in ((torch.bfloat16, ("out", "k_cache", "q")), (torch.float32, ("v_cache", "q"))):
            good = _tensors("cuda:0", hd=hd, dtype=dtype)[name]
            good["out"] = torch.zeros(good["q"].shape[0], good["q"].shape[1] * hd, dtype=dtype, device="cuda:0")
            for splits in (None, 0, 2):
                getattr(ops, name)(**good, n_splits=splits)
                for key in wrong:
                    with pytest.raises(ops.KernelError, match="alignment"):
                        getattr(ops, name)(**{**good, key: off(good[key])}, n_splits=splits)
