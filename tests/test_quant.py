"""CPU tests of the 8-bit latent cache and the attention over it: the oracle's
arithmetic and the refusals of the C ABI and of the Python entry points."""

import ctypes
import math

import pytest
import torch

from dsa_b200 import _native, quant
from oracle import quant as oq

P = ctypes.c_void_p


def kv_rows(n, seed, spread=12):
    g = torch.Generator().manual_seed(seed)
    kv = torch.randn(n, 576, generator=g) * torch.exp2(torch.randint(-spread, spread + 1, (n, 1), generator=g).float())
    return kv.bfloat16()


def angles(positions, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(positions, 32, generator=g) * 2 * math.pi
    return torch.cat([a.cos(), a.sin()], 1)


def test_oracle_codes_are_those_of_float8():
    x = torch.cat([torch.linspace(-448, 448, 20001), torch.randn(20000) * 2 ** -7, torch.tensor([0.0, -0.0, math.nan])])
    assert torch.equal(oq.e4m3(x.double()), x.to(torch.float8_e4m3fn).view(torch.uint8))
    every = torch.arange(256).to(torch.uint8)
    assert torch.equal(oq.value(every).nan_to_num(nan=1e9), every.view(torch.float8_e4m3fn).double().nan_to_num(nan=1e9))


@pytest.mark.parametrize("norm", [False, True])
def test_oracle_rows(norm):
    kv = kv_rows(40, 1)
    kv[3, :512] = 0
    kv[4, 7] = math.inf
    kv[5, 9] = math.nan
    w = (1 + 0.3 * torch.randn(512)).bfloat16() if norm else None
    code, scale, e = oq.write_rows(kv, w, 1e-6, torch.arange(40), angles(40))
    c = kv[:, :512].double()
    y = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-6) * w.double() if norm else c
    fine = [i for i in range(40) if i not in (4, 5)]
    # half a step of the codes, 2^-4 of a value or 2^-10 of the scale
    off = (oq.value(code) * scale[:, None] - y)[fine].abs()
    assert (off <= 2.0 ** -4 * y[fine].abs() + 2.0 ** -10 * scale[fine, None] + 1e-12).all()
    assert torch.isnan(oq.value(code)[4:6]).all() and (code[3] == 0).all() and (scale[3:6] == 1).all()
    # a rotation keeps the length of each pair
    pairs = kv[:, 512:].double().reshape(40, 2, 32).square().sum(1)
    assert torch.allclose(e.reshape(40, 2, 32).square().sum(1), pairs, rtol=1e-6)


def write_call(lib, kv=4096, row=1152, slots=16, n=2, norm=32, positions=64, table=128, most=7, cache=1 << 20, pages=3,
               status=None):
    return lib.dsa_latent_cache_write(P(kv), row, P(slots), n, P(norm), 1e-6, P(positions), P(table), most, 0, P(cache), pages,
                                      P(status), None)


@pytest.mark.parametrize("change,status", [
    (dict(n=-1), 1), (dict(n=0), 0), (dict(kv=None), 1), (dict(slots=None), 1), (dict(cache=None), 1), (dict(pages=-1), 1),
    (dict(row=1136), 1), (dict(positions=None), 1), (dict(table=None), 1), (dict(most=0), 1), (dict(kv=4104), 2),
    (dict(row=1160), 2), (dict(cache=(1 << 20) + 8), 2), (dict(norm=40), 2), (dict(slots=20), 2), (dict(positions=68), 2),
    (dict(table=132), 2), (dict(status=18), 2), (dict(kv=(1 << 20) + 3 * 41216 - 16), 7), (dict(kv=(1 << 20) - 2288), 7),
    (dict(slots=(1 << 20) + 8), 7), (dict(norm=(1 << 20) + 16), 7), (dict(positions=(1 << 20) - 8), 7),
    (dict(table=(1 << 20) - 1784), 7),
])
def test_write_c_abi_refuses_bad_arguments(change, status):
    assert write_call(_native.lib(), **change) == status


def read_call(lib, cache=1 << 20, pages=3, table=16, starts=64, cu=80, requests=2, max_pages=4, rows=5, ckv=1 << 21,
              ckv_row=1024, kpe=1 << 22, kpe_row=128, status=96):
    return lib.dsa_latent_cache_read(P(cache), pages, P(table), P(starts), P(cu), requests, max_pages, rows, P(ckv), ckv_row,
                                     P(kpe), kpe_row, P(status), None)


@pytest.mark.parametrize("change,status", [
    (dict(rows=-1), 1), (dict(rows=0), 0), (dict(requests=0), 0), (dict(requests=-1), 1), (dict(cache=None), 1),
    (dict(status=None), 1), (dict(pages=0), 1), (dict(max_pages=0), 1), (dict(ckv_row=1008), 1), (dict(kpe_row=112), 1),
    (dict(ckv=(1 << 21) + 8), 2), (dict(kpe_row=136), 2), (dict(cu=82), 2), (dict(cache=(1 << 20) + 8), 2),
    (dict(ckv=(1 << 20) + 3 * 41216 - 16), 7), (dict(kpe=(1 << 20) - 16), 7), (dict(kpe=(1 << 21) + 16), 7),
    (dict(table=(1 << 21) + 16), 7), (dict(cu=(1 << 22) + 4), 7),
])
def test_read_c_abi_refuses_bad_arguments(change, status):
    assert read_call(_native.lib(), **change) == status


def attend_call(lib, q=1 << 20, qp=1 << 21, cache=1 << 24, pages=3, lens=16, table=64, cu=128, requests=2, rows=3, heads=16, max_pages=4,
                out=1 << 22, lse=1 << 23, ws=1 << 28, nbytes=1 << 30):
    return lib.dsa_latent_attention_run(P(q), P(qp), P(cache), pages, P(lens), P(table), P(cu), requests, rows, heads, max_pages,
                                        0.1, P(out), P(lse), P(ws), nbytes, None)


@pytest.mark.parametrize("change,status", [
    (dict(requests=-1), 1), (dict(rows=-1), 1), (dict(rows=0), 0), (dict(requests=0), 0), (dict(heads=0), 1), (dict(heads=129), 1),
    (dict(requests=65537), 1), (dict(rows=(1 << 20) + 1), 1), (dict(q=None), 1), (dict(cache=None), 1), (dict(lens=None), 1),
    (dict(table=None), 1), (dict(cu=None), 1), (dict(ws=None), 1), (dict(out=None), 1), (dict(pages=0), 1), (dict(max_pages=0), 1),
    (dict(max_pages=(1 << 24) + 1), 1), (dict(max_pages=1 << 24, rows=1 << 12), 1), (dict(q=(1 << 20) + 8), 2), (dict(cache=(1 << 24) + 8), 2),
    (dict(out=(1 << 22) + 8), 2), (dict(lse=(1 << 23) + 2), 2), (dict(cu=130), 2), (dict(out=(1 << 24) + 3 * 41216 - 16), 7),
    (dict(out=(1 << 20) + 16), 7), (dict(out=(1 << 21) + 16), 7), (dict(lse=(1 << 22) + 16), 7), (dict(lse=16), 7), (dict(lse=136), 7),
    (dict(lse=(1 << 24) + 8), 7),
])
def test_attend_c_abi_refuses_bad_arguments(change, status):
    assert attend_call(_native.lib(), **change) == status


def sparse_call(lib, q=1 << 20, qp=1 << 21, cache=1 << 24, pages=3, idx=64, rows=3, heads=16, topk=8, out=1 << 22, lse=1 << 23,
                ws=1 << 28, nbytes=1 << 30):
    return lib.dsa_latent_sparse_attention_run(P(q), P(qp), P(cache), pages, P(idx), rows, heads, topk, 0.1, P(out), P(lse),
                                               P(ws), nbytes, None)


@pytest.mark.parametrize("change,status", [
    (dict(rows=-1), 1), (dict(rows=0), 0), (dict(heads=0), 1), (dict(heads=129), 1), (dict(topk=0), 1), (dict(topk=65537), 1),
    (dict(rows=(1 << 20) + 1, heads=1), 1), (dict(rows=(1 << 19) + 1, heads=17), 1), (dict(pages=0), 1), (dict(pages=1 << 25), 1),
    (dict(q=None), 1), (dict(idx=None), 1), (dict(qp=(1 << 21) + 8), 2), (dict(idx=66), 2), (dict(out=(1 << 24) + 16), 7),
    (dict(lse=64 + 92), 7), (dict(out=(1 << 20) + 32), 7),
])
def test_sparse_c_abi_refuses_bad_arguments(change, status):
    assert sparse_call(_native.lib(), **change) == status


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up: no launch may follow")
def test_output_in_place_of_the_queries_is_taken():
    assert attend_call(_native.lib(), out=1 << 20) not in (1, 2, 3, 7)
    assert sparse_call(_native.lib(), out=1 << 20) not in (1, 2, 3, 7)


def test_workspace_is_the_same_for_every_call():
    # without a GPU: two records of 32 rows for each of 160 SMs, and the groups of the largest call
    records, groups = 2 * 160 * 32 * (512 + 2) * 4, 2 * (2 ** 24 // 16 + 65536) * 4
    assert _native.lib().dsa_latent_attention_workspace_bytes() >= 256 + records * 148 // 160 + groups


def test_oracle_attention_is_softmax():
    """The oracle of dense and sparse rows against softmax over dequantised latents."""
    g = torch.Generator().manual_seed(1)
    cache = torch.zeros(3, quant.PAGE_BYTES, dtype=torch.uint8)
    codes, kpe, scales = oq.pieces(cache)
    codes[:] = torch.randn(codes.shape, generator=g).mul(100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    kpe[:] = torch.randn(kpe.shape, generator=g).bfloat16()
    scales[:] = torch.rand(scales.shape, generator=g) * 0.02
    qn, qp = torch.randn(2, 4, 512, generator=g).bfloat16(), torch.randn(2, 4, 64, generator=g).bfloat16()
    table = torch.tensor([[2, 0]])
    out, lse, bo, bl = oq.attend_reference(qn, qp, cache, torch.tensor([100]), table, torch.tensor([0, 2]), 0.05)
    lat = (codes.view(torch.float8_e4m3fn).double() * scales[..., None].double())
    k = torch.cat([lat[2], lat[0]])[:100], torch.cat([kpe[2], kpe[0]])[:100].double()
    for i, n in ((0, 99), (1, 100)):
        x = (qn[i].double() @ k[0][:n].T + qp[i].double() @ k[1][:n].T) * 0.05
        assert torch.allclose(out[i], torch.softmax(x, 1) @ k[0][:n], atol=1e-12)
        assert torch.allclose(lse[i], torch.logsumexp(x, 1) / math.log(2), atol=1e-12)
    assert (bo > 0).all() and (bo < 0.2).all() and (bl < 1e-2).all()
    picked = torch.cat([torch.arange(64) + 128, torch.full((7,), -1), torch.arange(36)])[None].int()
    so, sl, _, _ = oq.sparse_reference(qn[1:], qp[1:], cache, picked, 0.05)
    assert torch.allclose(so[0], out[1], atol=1e-12) and torch.allclose(sl[0], lse[1], atol=1e-12)


def test_entry_points_refuse_cpu_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        quant.write(kv_rows(2, 1), torch.zeros(2).long(), torch.zeros(1, quant.PAGE_BYTES, dtype=torch.uint8))
    with pytest.raises(ValueError, match="CUDA"):
        quant.read(torch.zeros(1, quant.PAGE_BYTES, dtype=torch.uint8), torch.zeros(1, 1).int(), torch.zeros(1).int(),
                   torch.zeros(2).int(), torch.zeros(1, 512).bfloat16(), torch.zeros(1, 64).bfloat16())
    rows = (torch.zeros(1, 16, 512).bfloat16(), torch.zeros(1, 16, 64).bfloat16(), torch.zeros(1, quant.PAGE_BYTES, dtype=torch.uint8))
    outs = torch.zeros(1, 16, 512).bfloat16(), torch.zeros(1, 16)
    with pytest.raises(ValueError, match="CUDA"):
        quant.attend(*rows, torch.zeros(1).int(), torch.zeros(1, 1).int(), None, 0.1, *outs)
    with pytest.raises(ValueError, match="CUDA"):
        quant.attend_sparse(*rows, torch.zeros(1, 2048).int(), 0.1, *outs)
