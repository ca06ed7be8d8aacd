"""What the calls over paged caches of 16, 8 and 4 bits refuse, before anything reaches the GPU."""
import ctypes as C
import importlib

import pytest
import torch

mynn = importlib.import_module("my-nn-engine_amd")

P16 = 0x10000  # an address that is never used: every call here is refused on the host


def append(**kw):
    a = dict(q_out=P16, q=P16, k=P16, v=P16, strides=(C.c_int64 * 9)(*[64] * 9), cos=P16, sin=P16, rows=8, position=None, kp=P16, vp=P16, ks=P16, vs=P16, kz=P16, vz=P16,
             table=P16, n_pages=4, pages=2, page_rows=32, past=P16, new=None, B=1, S=1, Hq=2, Hkv=1, D=64, dtype=mynn.F16, bits=4, group=64)
    a.update(kw)
    return mynn.lib().mynn_rope_append_paged(*a.values(), None)


def rows(**kw):
    a = dict(k=P16, v=P16, kp=P16, vp=P16, ks=P16, vs=P16, kz=P16, vz=P16, table=P16, n_pages=4, pages=2, page_rows=32, past=P16, new=None, B=1, S=1, Hkv=1, D=64,
             dtype=mynn.F16, bits=4, group=64)
    a.update(kw)
    return mynn.lib().mynn_kv_rows_paged(*a.values(), None)


def attend(**kw):
    a = dict(out=P16, q=P16, kp=P16, vp=P16, ks=P16, vs=P16, kz=P16, vz=P16, table=P16, n_pages=4, pages=2, page_rows=32, scale=1.0, causal=1, B=1, S=1, past=P16, new=None,
             Hq=2, Hkv=1, D=64, dtype=mynn.F16, group=64, ws=P16, ws_bytes=1 << 40, counters=None)
    a.update(kw)
    return mynn.lib().mynn_attention_paged_int4(*a.values(), None)


INVALID = [dict(kp=None), dict(vp=P16 + 8), dict(ks=None), dict(vs=P16 + 2), dict(kz=None), dict(vz=P16 + 1), dict(table=None), dict(past=None), dict(n_pages=0), dict(pages=0),
           dict(page_rows=48), dict(page_rows=16), dict(B=0), dict(S=-1), dict(Hkv=0)]
UNSUPPORTED = [dict(D=96), dict(D=256), dict(group=16), dict(group=128), dict(dtype=mynn.F32), dict(pages=1 << 20, page_rows=1 << 20)]


@pytest.mark.parametrize("call", [append, rows, attend])
@pytest.mark.parametrize("kw", INVALID + UNSUPPORTED, ids=str)
def test_common_refusals(call, kw):
    assert call(**kw) == (-1 if kw in INVALID else -2)
    assert mynn.lib().mynn_last_error()


@pytest.mark.parametrize("call,kw,code", [
    (append, dict(q=None), -1), (append, dict(q_out=None), -1), (append, dict(k=None), -1), (append, dict(strides=None), -1), (append, dict(cos=None), -1),
    (append, dict(rows=0), -1), (append, dict(bits=5), -1), (append, dict(q_out=P16 + 2), -1), (append, dict(B=1 << 20, S=1 << 20), -2),
    (rows, dict(k=None, v=None), -1), (rows, dict(v=P16 + 4), -1), (rows, dict(bits=3), -1), (rows, dict(B=1 << 20, S=1 << 20), -2),
    (attend, dict(q=None), -1), (attend, dict(out=P16 + 8), -1), (attend, dict(Hq=3, Hkv=2), -1), (attend, dict(Hq=1 << 15, S=1 << 20), -2),
    (attend, dict(pages=64, ws=None), -1), (attend, dict(pages=64, ws_bytes=64), -1), (attend, dict(pages=64, ws=P16 + 8), -1), (attend, dict(counters=P16 + 2), -1),
    (attend, dict(pages=64, S=64, ws=None), -1), (attend, dict(B=1 << 24, S=64), -2), (attend, dict(B=1 << 28, pages=1 << 20), -2), (append, dict(B=1 << 24, S=64), -2),
    (rows, dict(B=1 << 24, S=64), -2),
], ids=str)
def test_refusals_of_each(call, kw, code):
    assert call(**kw) == code and mynn.lib().mynn_last_error()


def pools(bits=4, n=4, H=1, P=32, D=64, group=64, t=torch.float16):
    lead = (n, H, P)
    if bits == 16:
        return [torch.zeros(lead + (D,), dtype=t) for _ in range(2)]
    if bits == 8:
        return [torch.zeros(lead + (D,), dtype=torch.int8) for _ in range(2)] + [torch.zeros(lead, dtype=t) for _ in range(2)]
    return [torch.zeros(lead + (D // 2,), dtype=torch.uint8) for _ in range(2)] + [torch.zeros(lead + (D // group,), dtype=x) for x in (t, t, torch.uint8, torch.uint8)]


def test_the_python_calls_refuse_what_does_not_fit_together():
    table, past = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    k = torch.zeros(1, 1, 1, 64, dtype=torch.float16)
    cos = torch.zeros(8, 64, dtype=torch.float16)
    good = pools()
    bad_pools = [good[:5], good[:3], [good[0].char()] + good[1:], good[:2] + [good[2].float()] + good[3:], good[:4] + [good[4][..., :0]] + good[5:],
                 [good[0][:2]] + good[1:], good[:2] + [good[2].bfloat16()] + good[3:], [t[0] for t in good]]
    for bad in bad_pools:
        with pytest.raises(mynn.MynnError):
            mynn.rope_append_paged(q, k, k, cos, cos, bad, table, past)
        with pytest.raises(mynn.MynnError):
            mynn.attention_paged_int4(q, bad, table, 1.0, past)
        with pytest.raises(mynn.MynnError):
            mynn.kv_rows_paged(bad, table, past, 1)
    # (operands of the CPU are refused by the pointer check, at the last)
    for call in (lambda: mynn.rope_append_paged(q, k, k, cos, cos, good, table, past), lambda: mynn.attention_paged_int4(q, good, table, 1.0, past),
                 lambda: mynn.kv_rows_paged(good, table, past, 1)):
        with pytest.raises(AssertionError):
            call()


def test_four_bit_buffers_of_a_pool_ask_for_groups_that_divide_a_row():
    pool = mynn.KvPool(2, 32)
    for kw in (dict(kv_int4_group=16), dict(kv_int4_group=128), dict(kv_int4_group=64, kv_int8=True)):
        with pytest.raises(mynn.MynnError):
            pool.buffers(1, 1, 64, torch.float16, **kw)
    pool.close()


def test_workspaces_ask_for_what_a_call_needs():
    size = mynn.lib().mynn_attention_paged_int4_workspace_bytes
    assert size(0, 1, 8, 32, 8, 2, 64) == 0 and size(1, 1, 8, 32, 1, 2, 64) == 0
    for S in (1, 4, 5, 64, 500):
        last = 0
        for pages in (1, 8, 64, 512):
            need = size(2, S, pages, 64, 8, 2, 128)
            assert last <= need < 256 << 20  # (more keys, more parts; they end with the device's compute units)
            last = need
    header = open(mynn.CSRC + "/../../include/mynn_hip.h").read()
    assert "#define MYNN_PAGED_INT4_COUNTERS %d" % (mynn.PAGED_INT4_COUNTER_BYTES // 4) in header
