"""What the operators of the 4-bit cache refuse before anything is launched (no GPU: tensors without memory, null pointers)."""
import pytest
import torch

from kvcm_amd import ops

NH, NKV, HD, PAGE, PAGES, T = 4, 2, 64, 32, 9, 3
BF, F32, I32, U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8


def e(*shape, dtype=I32):
    return torch.empty(shape, dtype=dtype, device="meta")


def cache(pages=PAGES, nkv=NKV, hd=HD, page=PAGE, dtype=U8):
    return e(pages, nkv, page // 16, 16 * (hd + 8), dtype=dtype)


@pytest.fixture(autouse=True)
def no_gpu(monkeypatch):
    monkeypatch.setattr(ops, "_one_gpu", lambda *tensors: [0] * len(tensors))
    monkeypatch.setattr(ops, "_stream", lambda: 0)


def store(**kw):
    a = dict(qkv=e(T, (NH + 2 * NKV) * HD, dtype=BF), nh=NH, nkv=NKV, hd=HD, cache=cache(), slots=e(T)) | kw
    ops.rope_cache4(**a)


def read(**kw):
    a = dict(cache=cache(), slots=e(T), k=e(T, NKV * HD, dtype=BF), v=e(T, NKV * HD, dtype=BF)) | kw
    ops.cache4_rows(**a)


def decode(**kw):
    a = dict(q=e(T, NH * HD, dtype=BF), out=e(T, NH * HD, dtype=BF), cache=cache(), tables=e(2, 4), table_stride=4, row_seq=e(T), ctx_lens=e(T),
             nh=NH, nkv=NKV, hd=HD, scale=0.125, max_context=100) | kw
    ops.attention_decode4(**a)


def prefill(**kw):
    a = dict(q=e(T, NH * HD, dtype=BF), out=e(T, NH * HD, dtype=BF), cache=cache(), tables=e(2, 4), table_stride=4, run_start=e(3), seq_start=e(2),
             num_seqs=2, max_run=2, nh=NH, nkv=NKV, hd=HD, scale=0.125) | kw
    ops.attention_prefill4(**a)


@pytest.mark.parametrize("call", (store, read, decode, prefill))
def test_what_is_no_cache_is_refused(call):
    for bad in (cache(dtype=torch.int8), e(PAGES, NKV, 16 * (HD + 8), dtype=U8), e(PAGES, NKV, 2, 16 * (HD + 8) + 16, dtype=U8),
                e(PAGES, 2, NKV, 16 * (HD + 8), dtype=U8).transpose(1, 2)[:, :, :1].expand(PAGES, NKV, 2, -1),
                cache(hd=48), cache(pages=2 ** 26, page=32)):
        with pytest.raises(ValueError, match="cache"):
            call(cache=bad)
    if call is not read:
        for bad in (cache(nkv=1), cache(hd=128)):
            with pytest.raises(ValueError, match="cache"):
                call(cache=bad)


@pytest.mark.parametrize("bad, match", (
    (dict(qkv=e(T, (NH + 2 * NKV) * HD - 1, dtype=BF)), "qkv"), (dict(qkv=e(T, (NH + 2 * NKV) * HD, dtype=torch.float16)), "qkv"),
    (dict(qkv=e((NH + 2 * NKV) * HD, T, dtype=BF).T), "qkv"), (dict(qkv=e(1, (NH + 2 * NKV) * HD, dtype=BF).expand(T, -1)), "qkv"),
    (dict(slots=e(T - 1)), "slots"), (dict(slots=e(T, dtype=torch.int64)), "slots"), (dict(rows=T + 1), "qkv"), (dict(rows=-1), "qkv"), (dict(nh=3), "heads"),
    (dict(cos_sin=e(T, HD // 2, 2, dtype=BF)), "cos_sin"), (dict(cos_sin=e(T - 1, HD // 2, 2, dtype=F32)), "cos_sin"),
    (dict(q_out=e(T, NH * HD, dtype=BF)), "q_out"),
    (dict(cos_sin=e(T, HD // 2, 2, dtype=F32), q_out=e(T, NH * HD, dtype=F32)), "q_out"),
    (dict(cos_sin=e(T, HD // 2, 2, dtype=F32), q_out=e(T, NH * HD - 8, dtype=BF)), "q_out")))
def test_store_refuses(bad, match):
    with pytest.raises(ValueError, match=match):
        store(**bad)


@pytest.mark.parametrize("bad, match", (
    (dict(k=e(T, NKV * HD - 1, dtype=BF)), "k must"), (dict(v=e(T, NKV * HD, dtype=F32)), "v must"), (dict(k=e(T - 1, NKV * HD, dtype=BF)), "k must"),
    (dict(slots=e(T, dtype=torch.int64)), "slots"), (dict(k=e(T, NKV * HD, dtype=torch.float16)), "k must")))
def test_read_refuses(bad, match):
    with pytest.raises(ValueError, match=match):
        read(**bad)


ATTENTION = ((dict(q=e(T, NH * HD - 1, dtype=BF)), "q must"), (dict(out=e(T, NH * HD, dtype=F32)), "out must"), (dict(q=e(T, NH * HD, dtype=torch.float16)), "q must"),
             (dict(out=e(1, NH * HD, dtype=BF).expand(T, -1)), "out must"), (dict(rows=T + 1), "q must"), (dict(table_stride=0), "table_stride"), (dict(window=-1), "window"),
             (dict(nh=5), "heads"), (dict(max_context=-1), "max_context"), (dict(tables=e(2, 4, dtype=torch.int64)), "tables"))


@pytest.mark.parametrize("bad, match", ATTENTION + (
    (dict(row_seq=e(T - 1)), "row_seq"), (dict(ctx_lens=e(T - 1)), "ctx_lens"), (dict(tables=e(3)), "tables")))
def test_decode_refuses(bad, match):
    with pytest.raises(ValueError, match=match):
        decode(**bad)


@pytest.mark.parametrize("bad, match", ATTENTION + (
    (dict(run_start=e(2)), "run_start"), (dict(seq_start=e(1)), "seq_start"), (dict(tables=e(7)), "tables"), (dict(max_run=-1), "max_run"), (dict(num_seqs=-1), "num_seqs")))
def test_prefill_refuses(bad, match):
    with pytest.raises(ValueError, match=match):
        prefill(**bad)


def test_scratch_is_checked_and_a_recorded_step_brings_it(monkeypatch):
    monkeypatch.setattr(ops, "attention_decode4_scratch", lambda *a: 100)
    monkeypatch.setattr(ops, "attention_prefill4_scratch", lambda *a: 100)
    for call in (decode, prefill):
        with pytest.raises(ValueError, match="100 floats"):
            call(scratch=e(99, dtype=F32))
        with pytest.raises(ValueError, match="float32"):
            call(scratch=e(100, dtype=torch.float64))
        monkeypatch.setattr(ops, "_recording", object())
        with pytest.raises(ValueError, match="bring its scratch"):
            call()
        monkeypatch.setattr(ops, "_recording", None)


def test_the_c_entries_refuse_what_their_kernels_do_not_take():
    lib = ops.lib()
    said = lambda: lib.kvcm_hip_last_error().decode()
    p = 4096      # never read: every call is refused on the host
    assert lib.kvcm_rope_cache4(p, 1, 512, 0, 0, p, p, 0, 3, 4, 2, 48, 9, 32, 0) == -1 and "head_dim 48" in said()
    assert lib.kvcm_rope_cache4(p, 1, 511, 0, 0, p, p, 0, 3, 4, 2, 64, 9, 32, 0) == -1 and "511" in said()
    assert lib.kvcm_rope_cache4(p, 1, 512, 0, 0, p, p, 0, 3, 4, 2, 64, 9, 24, 0) == -1 and "24 tokens" in said()
    assert lib.kvcm_rope_cache4(p, 7, 512, 0, 0, p, p, 0, 3, 4, 2, 64, 9, 32, 0) == -1 and "dtype" in said()
    assert lib.kvcm_rope_cache4(0, 1, 512, 0, 0, p, p, 0, 3, 4, 2, 64, 9, 32, 0) == -1 and "null" in said()
    assert lib.kvcm_rope_cache4(p, 1, 512, 0, 256, p, p, p, 3, 4, 2, 64, 9, 32, 0) == -1 and "null" in said()
    assert lib.kvcm_rope_cache4(p, 1, 512, 0, 0, p, p, 0, 3, 4, 2, 64, 2 ** 26, 32, 0) == -1 and "pages" in said()
    assert lib.kvcm_cache4_rows(p, p, p, 128, p, 127, 1, 3, 2, 64, 9, 32, 0) == -1 and "127" in said()
    assert lib.kvcm_cache4_rows(p, p, 0, 128, p, 128, 1, 3, 2, 64, 9, 32, 0) == -1 and "null" in said()
    dec = lambda **k: lib.kvcm_attention_decode4(*(dict(q=p, dt=1, qs=256, out=p, os=256, c=p, tab=p, stride=4, seqs=2, rs=p, cl=p, T=3, nh=4, nkv=2, hd=64, pages=9,
                                                       page=32, scale=0.1, window=0, mc=100, scr=0, n=0, stream=0) | k).values())
    pre = lambda **k: lib.kvcm_attention_prefill4(*(dict(q=p, dt=1, qs=256, out=p, os=256, c=p, tab=p, stride=4, rs=p, ss=p, seqs=2, mr=2, T=3, nh=4, nkv=2, hd=64,
                                                        pages=9, page=32, scale=0.1, window=0, mc=100, scr=0, n=0, stream=0) | k).values())
    for call in (dec, pre):
        for bad, word in ((dict(hd=80), "head_dim 80"), (dict(nh=5), "heads 5"), (dict(page=8), "8 tokens"), (dict(dt=2), "dtype"), (dict(qs=255), "255"),
                          (dict(window=-1), "window"), (dict(stride=0), "tables"), (dict(q=0), "null"), (dict(c=0), "null"), (dict(T=-1), "rows"),
                          (dict(stride=2 ** 27), "tables")):
            assert call(**bad) == -1 and word in said(), (bad, said())
        assert call(T=0) == 0


def test_the_shape_of_a_cache():
    assert ops.cache4_shape(7, 4, 64, 32) == (7, 4, 2, 1152)
    assert ops.cache4_supported(32, 4, 64, BF) and ops.cache4_supported(32, 8, 128, F32, 64)
    assert not ops.cache4_supported(32, 4, 64, torch.float16) and not ops.cache4_supported(32, 5, 64, BF) and not ops.cache4_supported(32, 4, 96, BF)
    assert not ops.cache4_supported(32, 4, 64, BF, 8)
    for bad in ((0, 4, 64, 16), (7, 4, 48, 16), (7, 4, 64, 24), (7, 0, 64, 16)):
        with pytest.raises(ValueError, match="4-bit cache"):
            ops.cache4_shape(*bad)


def test_numbers_that_do_not_fit_are_refused():
    for call in (decode, prefill):
        for bad in (dict(window=2 ** 31), dict(max_context=2 ** 32 + 5)):
            with pytest.raises(ValueError, match="fit 32 bits"):
                call(**bad)
    with pytest.raises(ValueError, match="fit 32 bits"):
        prefill(max_run=2 ** 31)
    said, p, lib = lambda: ops.lib().kvcm_hip_last_error().decode(), 4096, ops.lib()
    assert lib.kvcm_rope_cache4(p, 1, 512, 0, 0, p, p, 0, 2 ** 28, 4, 2, 64, 9, 32, 0) == -1 and "too many" in said()
    assert lib.kvcm_cache4_rows(p, p, p, 512, p, 512, 1, 2 ** 28, 8, 64, 9, 32, 0) == -1 and "too many" in said()
    assert lib.kvcm_attention_decode4(p, 1, 256, p, 256, p, p, 4, 2, p, p, 70000, 4, 2, 64, 9, 32, 0.1, 0, 100, 0, 0, 0) == -1 and "70000" in said()
    assert lib.kvcm_attention_prefill4(p, 1, 256, p, 256, p, p, 4, p, p, 2, 2 ** 30, 2 ** 30, 4, 2, 64, 9, 32, 0.1, 0, 100, 0, 0, 0) == -1 and "workgroups" in said()
    assert lib.kvcm_attention_decode4_scratch(1, 4, 2, 64, 2 ** 31 - 1, 2 ** 31 - 1) >= 0
    assert lib.kvcm_rope_cache4(p, 1, 4096, 0, 0, p, p, 0, 2 ** 25, 8, 4, 256, 9, 32, 0) == -1 and "too many" in said()      # 2^32 threads and more
    assert lib.kvcm_cache4_rows(p, p, p, 1024, p, 1024, 1, 2 ** 25, 4, 256, 9, 32, 0) == -1 and "too many" in said()
    assert lib.kvcm_attention_prefill4(p, 1, 8192, p, 8192, p, p, 2 ** 22, p, p, 1, 2 ** 24, 2 ** 24, 32, 32, 256, 9, 32, 0.1, 0, 2 ** 24, 0, 0, 0) == -1 and "workgroups" in said()


def test_operands_elsewhere_are_refused(monkeypatch):
    monkeypatch.undo()
    for call in (store, read, decode, prefill):
        with pytest.raises(ValueError, match="GPU"):
            call()


@pytest.mark.parametrize("nh, nkv, hd", ((32, 4, 64), (32, 8, 128), (16, 2, 256), (3, 1, 32)))
def test_scratch_of_any_size_is_bounded(nh, nkv, hd):
    """Parts fill the chip, whatever the contexts: scratch stays a small part of what the cache takes, and grows with nothing but the rows."""
    for rows in (1, 3, 17, 64, 500, 5000):
        for ctx in (0, 1, 100, 513, 4096, 33000, 2 ** 20, 2 ** 30):
            for window in (0, 1, 4096):
                floats = ops.attention_decode4_scratch(rows, nh, nkv, hd, ctx, window)
                assert 0 <= floats <= (1536 // nkv + 3 * rows) * nh * (hd + 2), (rows, ctx, window)
                assert ctx > 256 or floats == 0
                runs = ops.attention_prefill4_scratch(rows, nh, nkv, hd, ctx, rows, 1, window)
                assert 0 <= runs <= rows * nh * (1536 // nkv + 2) * (hd + 2)


def test_scratch_goes_by_values():
    """Sizes may be anything that counts, and what they come to is never a former call's."""
    size = torch.tensor(100)
    assert ops.attention_decode4_scratch(1, 32, 8, 128, size) == 0
    size += 30000
    assert ops.attention_decode4_scratch(1, 32, 8, 128, size) == ops.attention_decode4_scratch(1, 32, 8, 128, 30100) > 0


def test_queries_written_over_rows_that_are_still_read_are_refused(monkeypatch):
    monkeypatch.setattr(ops, "_one_gpu", lambda *tensors: [0 if t is None else t.data_ptr() for t in tensors])
    monkeypatch.setattr(ops, "_call", lambda *args: None)
    wide = (NH + 2 * NKV) * HD
    for dtype in (BF, F32):
        held = torch.zeros(T + 2, wide + NH * HD + 7, dtype=dtype)
        rest = dict(slots=torch.zeros(T, dtype=I32), cos_sin=torch.zeros(T, HD // 2, 2), cache=torch.zeros(ops.cache4_shape(PAGES, NKV, HD, PAGE), dtype=U8), rows=T)
        rows, behind = held[:T, :wide], held[:T, NH * HD + 7:]
        store(qkv=rows, q_out=rows[:, :NH * HD], **rest)
        store(qkv=rows, q_out=rows, **rest)
        store(qkv=rows, q_out=held[:T, wide:], **rest)
        store(qkv=rows, q_out=held[:T, wide + 7:], **rest)
        store(qkv=behind, q_out=held[:T, :NH * HD], **rest)
        store(qkv=behind, q_out=held[:T, 7:], **rest)
        store(qkv=rows, q_out=torch.zeros(T, NH * HD, dtype=dtype), **rest)
        store(qkv=rows, q_out=held.view(-1)[:T * NH * HD].view(T, -1)[:1], **rest | dict(rows=1))
        for bad in (rows[:, 1:], rows[:, HD:], held[1:T + 1, :wide], held[:T, wide - 1:], held.view(-1)[:T * NH * HD].view(T, -1), held[:T, 7:]):
            with pytest.raises(ValueError, match="q_out must be the rows"):
                store(qkv=rows, q_out=bad, **rest)
        with pytest.raises(ValueError, match="q_out must be the rows"):
            store(qkv=behind, q_out=held[:T, 8:], **rest)


@pytest.mark.parametrize("call, bad", (
    (decode, dict(tables=e(2 ** 32 + 4), table_stride=2 ** 32 + 4)), (decode, dict(tables=e(2 ** 31), table_stride=2 ** 31)), (decode, dict(tables=e(2 ** 32 + 2), table_stride=1)),
    (prefill, dict(num_seqs=2 ** 32 + 2, run_start=e(2 ** 32 + 3), seq_start=e(2 ** 32 + 2), tables=e(2 ** 34 + 8))),
    (decode, dict(q=e(2 ** 32 + 3, NH * HD, dtype=BF), out=e(2 ** 32 + 3, NH * HD, dtype=BF), row_seq=e(2 ** 32 + 3), ctx_lens=e(2 ** 32 + 3))),
    (prefill, dict(q=e(2 ** 32 + 3, NH * HD, dtype=BF), out=e(2 ** 32 + 3, NH * HD, dtype=BF))),
    (store, dict(qkv=e(2 ** 32 + 3, (NH + 2 * NKV) * HD, dtype=BF), slots=e(2 ** 32 + 3))),
    (read, dict(slots=e(2 ** 32 + 3), k=e(2 ** 32 + 3, NKV * HD, dtype=BF), v=e(2 ** 32 + 3, NKV * HD, dtype=BF))),
    (decode, dict(nh=2 ** 32 + NH, q=e(1, (2 ** 32 + NH) * HD, dtype=BF), out=e(1, (2 ** 32 + NH) * HD, dtype=BF))),
    (store, dict(nh=2 ** 32 + NH, qkv=e(1, (2 ** 32 + NH + 2 * NKV) * HD, dtype=BF)))))
def test_counts_that_a_c_int_would_cut_are_refused(call, bad, monkeypatch):
    """Numbers that end in a small one where 32 bits are kept of them: none of them reaches the library."""
    monkeypatch.setattr(ops, "_call", lambda *args: pytest.fail(f"launched with {args}"))
    with pytest.raises(ValueError, match="32 bits|rows of their own"):
        call(**bad)
