"""Arguments that the 4-bit KV cache calls refuse, before any GPU work."""
import pytest

import swiftlet_b200 as swl

P = 1 << 20  # an aligned address that no refused call touches


def cache(**kw):
    d = dict(pages=P, page_table=P, table_stride=4, num_pages=8, page_size=64, kv_heads=2, head_dim=256, group=64)
    d.update(kw)
    return swl.swl_kv4_cache(**d)


def batch(**kw):
    d = dict(start=P, lens=P, nseq=1, total=1, max_new=1, max_len=100, status=None)
    d.update(kw)
    return swl.swl_kv4_batch(**d)


def refused(code, f):
    with pytest.raises(swl.SwiftletError) as e:
        f()
    assert e.value.code == code, str(e.value)


def attend(c=None, b=None, heads=16, **kw):
    d = dict(scale=0.1, d_work=P, work_bytes=1 << 40)
    d.update(kw)
    q, out = d.pop("q", P), d.pop("out", 2 * P)
    return lambda: swl.kv4_attention_device(c or cache(), b or batch(), heads, q, out, **d)


def evict(c=None, b=None, keep=50, **kw):
    d = dict(d_weights=P, weights_stride=100, d_dst_table=2 * P, dst_stride=4, d_new_lens=2 * P, d_kept=P, kept_stride=50)
    d.update(kw)
    return lambda: swl.kv4_evict_device(c or cache(), b or batch(), keep, **d)


@pytest.mark.parametrize("kw,code", [
    (dict(pages=None), swl.SWL_ERR_INVALID), (dict(page_table=None), swl.SWL_ERR_INVALID),
    (dict(pages=P + 8), swl.SWL_ERR_INVALID), (dict(num_pages=0), swl.SWL_ERR_INVALID),
    (dict(kv_heads=0), swl.SWL_ERR_INVALID), (dict(table_stride=0), swl.SWL_ERR_INVALID),
    (dict(head_dim=96), swl.SWL_ERR_UNSUPPORTED), (dict(group=32), swl.SWL_ERR_UNSUPPORTED),
    (dict(head_dim=64, group=128), swl.SWL_ERR_UNSUPPORTED), (dict(page_size=48), swl.SWL_ERR_UNSUPPORTED),
    (dict(page_size=256), swl.SWL_ERR_UNSUPPORTED)])
def test_cache(kw, code):
    c = cache(**kw)
    refused(code, lambda: swl.kv4_append_device(c, batch(), P, P))
    refused(code, lambda: swl.kv4_read_device(c, batch(), P, P))
    refused(code, attend(c))
    refused(code, evict(c))
    refused(code, lambda: swl.kv4_attention_workspace(c, batch(), 16))
    refused(code, lambda: swl.kv4_evict_workspace(c, batch(), 5))


@pytest.mark.parametrize("kw,code", [
    (dict(nseq=-1), swl.SWL_ERR_INVALID), (dict(total=-1), swl.SWL_ERR_INVALID), (dict(max_len=-1), swl.SWL_ERR_INVALID),
    (dict(lens=None), swl.SWL_ERR_INVALID), (dict(lens=P + 2), swl.SWL_ERR_INVALID), (dict(status=P + 1), swl.SWL_ERR_INVALID),
    (dict(max_len=257), swl.SWL_ERR_CAPACITY)])
def test_batch(kw, code):
    b = batch(**kw)
    refused(code, lambda: swl.kv4_append_device(cache(), b, P, P))
    refused(code, attend(b=b))
    refused(code, evict(b=b))


def test_tokens():
    refused(swl.SWL_ERR_INVALID, lambda: swl.kv4_append_device(cache(), batch(start=None), P, P))
    refused(swl.SWL_ERR_UNSUPPORTED, lambda: swl.kv4_append_device(cache(), batch(), P, P, dtype=3))
    refused(swl.SWL_ERR_INVALID, lambda: swl.kv4_append_device(cache(), batch(), 0, P))
    refused(swl.SWL_ERR_INVALID, lambda: swl.kv4_read_device(cache(), batch(), P, P + 2))
    refused(swl.SWL_ERR_INVALID, lambda: swl.kv4_append_device(cache(), batch(), P, P, k_strides=(-1, 256)))
    refused(swl.SWL_ERR_INVALID, lambda: swl.kv4_append_device(cache(), batch(), P, P, d_weights=P, weights_stride=99))


def test_attention():
    refused(swl.SWL_ERR_INVALID, attend(heads=15))
    refused(swl.SWL_ERR_INVALID, attend(heads=0))
    refused(swl.SWL_ERR_UNSUPPORTED, attend(heads=130))
    refused(swl.SWL_ERR_INVALID, attend(scale=float("nan")))
    refused(swl.SWL_ERR_INVALID, attend(q=0))
    refused(swl.SWL_ERR_INVALID, attend(out=P))
    refused(swl.SWL_ERR_INVALID, attend(d_gate=2 * P))
    refused(swl.SWL_ERR_INVALID, attend(d_weights=P, weights_stride=99))
    refused(swl.SWL_ERR_CAPACITY, attend(work_bytes=0))
    refused(swl.SWL_ERR_INVALID, attend(d_work=P + 4))
    refused(swl.SWL_ERR_UNSUPPORTED, attend(dtype=-1))


def test_evict():
    refused(swl.SWL_ERR_INVALID, evict(keep=-1))
    refused(swl.SWL_ERR_INVALID, evict(first=30, recent=21))
    refused(swl.SWL_ERR_INVALID, evict(d_weights=0))
    refused(swl.SWL_ERR_INVALID, evict(weights_stride=99))
    refused(swl.SWL_ERR_INVALID, evict(kept_stride=49))
    refused(swl.SWL_ERR_INVALID, evict(d_new_weights=2 * P, new_weights_stride=49))
    refused(swl.SWL_ERR_INVALID, evict(d_new_weights=P, new_weights_stride=50))
    refused(swl.SWL_ERR_INVALID, evict(d_new_lens=P))
    refused(swl.SWL_ERR_INVALID, evict(d_dst_table=P))
    refused(swl.SWL_ERR_CAPACITY, evict(keep=100, kept_stride=100, dst_stride=1))
    refused(swl.SWL_ERR_CAPACITY, evict(d_kept=0))


def test_empty_batches_do_nothing():
    for b in (batch(nseq=0, total=0), batch(total=0)):
        swl.kv4_append_device(cache(), b, P, P)
        swl.kv4_read_device(cache(), b, P, P)
        attend(b=b)()
    evict(b=batch(nseq=0))()


def test_page_bytes():
    assert swl.kv4_page_bytes(2, 256, 64, 64) == 2 * 2 * 64 * (128 + 16)
    assert swl.kv4_page_bytes(8, 64, 64, 128) == 8 * 2 * 128 * (32 + 4)
    refused(swl.SWL_ERR_UNSUPPORTED, lambda: swl.kv4_page_bytes(2, 80, 64, 64))


def test_bounds_near_the_end_of_32_bits():
    """Bounds that tile and row counts could not be rounded up from."""
    c = cache(table_stride=1 << 26)
    for kw in (dict(max_len=2 ** 31 - 1), dict(max_len=2 ** 31 - 4095), dict(total=2 ** 31 - 1), dict(total=2 ** 31 - 4095)):
        b = batch(**kw)
        refused(swl.SWL_ERR_UNSUPPORTED, lambda: swl.kv4_append_device(c, b, P, P))
        refused(swl.SWL_ERR_UNSUPPORTED, lambda: swl.kv4_read_device(c, b, P, P))
        refused(swl.SWL_ERR_UNSUPPORTED, lambda: swl.kv4_attention_workspace(c, b, 16))
        refused(swl.SWL_ERR_UNSUPPORTED, attend(c, b))
        refused(swl.SWL_ERR_UNSUPPORTED, evict(c, b))
        refused(swl.SWL_ERR_UNSUPPORTED, lambda: swl.kv4_evict_workspace(c, b, 5))
    b = batch(max_len=2 ** 31 - 4096, total=2 ** 31 - 4096)
    assert swl.kv4_attention_workspace(c, b, 16) > 0 and swl.kv4_evict_workspace(c, b, 5) == 2 * 5 * 4
