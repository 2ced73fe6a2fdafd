"""What the operators on the paged 8-bit cache refuse.  Descriptors are checked before the context, so none of this needs a
GPU: a descriptor with nothing wrong fails with "null context"."""
import ctypes as C

import pytest

import tachyon_b200 as tb
from tachyon_b200 import _lib, build

AT = 1 << 20  # stands for a device address: never followed, the context is missing


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def call(lib, name, args):
    status = getattr(lib, name)(None, None if args is None else C.byref(args))
    return status, lib.tb_last_error().decode()


def pages(**change):
    return tb.Pages(**(dict(k=AT, v=AT, k_scale=AT, v_scale=AT, table=AT, pages=100, page=16, kv_heads=2, head_dim=128, requests=3, width=7) | change))


def plan(**change):
    return tb.PagePlan(**(dict(lengths=AT, fresh=AT, lengths_out=AT, table=AT, free_pages=AT, free_count=AT, free_count_out=AT, starts=AT, slots=AT, positions=None,
                               refused=AT, scratch=AT, requests=3, width=7, page=16, pages=100, max_tokens=9) | change))


def rows(cache=None, **change):
    return tb.CacheRows(**(dict(cache=cache or pages(), k=AT, v=AT, dtype=tb.F32, token_stride=256, head_stride=128, slots=AT, tokens=5) | change))


def attend(cache=None, **change):
    return tb.PagedAttend(**(dict(cache=cache or pages(), q=AT, q_dtype=tb.F16, q_stride=1024, starts=AT, lengths=AT, tokens=5, heads=8, most=2, window=0, scale=1.0,
                                  out=AT, out_dtype=tb.F16, out_stride=1024, scratch=AT, scratch_bytes=1 << 30) | change))


def logits(**change):
    return tb.Logits(**(dict(logits=AT, out=AT, dtype=tb.F32, rows=2, vocab=100, stride=100, out_stride=100, history=AT, history_stride=9, prompt=AT, total=AT,
                             repetition=AT, frequency=AT, presence=AT, bias_token=AT, bias=AT, bias_count=AT, bias_stride=4, allowed=AT, mask_of=None, allowed_stride=4,
                             masks=2) | change))


GOOD = {"tb_page_plan": plan, "tb_cache_append_q8": rows, "tb_cache_read_q8": rows, "tb_attend_paged_q8": attend, "tb_prefill_paged_q8": attend, "tb_logits_adjust": logits}


@pytest.mark.parametrize("name", GOOD)
def test_a_good_descriptor_only_lacks_the_context(lib, name):
    assert call(lib, name, GOOD[name]()) == (3, "null context")
    status, text = call(lib, name, None)
    assert status == 3 and "null descriptor" in text


@pytest.mark.parametrize("change", [{"k": None}, {"v_scale": None}, {"page": 48}, {"page": 0}, {"page": 8}, {"pages": 0}, {"kv_heads": 0}, {"kv_heads": 2000}, {"k": AT + 8},
                                    {"pages": 1 << 28}])
@pytest.mark.parametrize("name", ["tb_cache_append_q8", "tb_cache_read_q8", "tb_attend_paged_q8", "tb_prefill_paged_q8"])
def test_a_bad_cache(lib, name, change):
    status, text = call(lib, name, GOOD[name](pages(**change)))
    assert status == 3 and text.startswith(name) and "null context" not in text
    assert call(lib, name, GOOD[name](pages(head_dim=96)))[0] == 9


@pytest.mark.parametrize("change", [{"lengths": None}, {"fresh": None}, {"table": None}, {"refused": None}, {"scratch": None}, {"slots": None}, {"page": 17}, {"page": 0},
                                    {"requests": 0}, {"requests": 8193}, {"width": 0}, {"width": 1 << 28}, {"pages": 0}, {"pages": 1 << 28}, {"max_tokens": 1 << 31},
                                    {"starts": AT + 2}])
def test_a_bad_plan(lib, change):
    status, text = call(lib, "tb_page_plan", plan(**change))
    assert status == 3 and text.startswith("tb_page_plan")


@pytest.mark.parametrize("change", [{"k": None}, {"slots": None}, {"dtype": 2}, {"token_stride": 252}, {"head_stride": 4}, {"v": AT + 8}, {"slots": AT + 1}, {"tokens": 1 << 31}])
@pytest.mark.parametrize("name", ["tb_cache_append_q8", "tb_cache_read_q8"])
def test_bad_rows(lib, name, change):
    status, text = call(lib, name, rows(**change))
    assert status == 3 and text.startswith(name)


@pytest.mark.parametrize("change", [{"q": None}, {"out": None}, {"lengths": None}, {"q_dtype": 7}, {"out_dtype": -1}, {"heads": 0}, {"heads": 7}, {"most": 0}, {"scale": 0.0},
                                    {"scale": -1.0}, {"scale": float("nan")}, {"scale": float("inf")}, {"q_stride": 1020}, {"q_stride": 512}, {"out_stride": 1016},
                                    {"q": AT + 2}, {"starts": None}, {"tokens": 1 << 31}, {"most": 1 << 30}])
@pytest.mark.parametrize("name", ["tb_attend_paged_q8", "tb_prefill_paged_q8"])
def test_a_bad_attention(lib, name, change):
    status, text = call(lib, name, attend(**change))
    assert status == 3 and text.startswith(name)


def test_attention_shapes_without_a_kernel(lib):
    assert call(lib, "tb_attend_paged_q8", attend(heads=130, q_stride=1 << 20, out_stride=1 << 20))[0] == 9  # 65 query heads to a key-value head
    status, text = call(lib, "tb_attend_paged_q8", attend(most=17))  # 68 query rows
    assert status == 9 and "tb_prefill_paged_q8" in text
    assert call(lib, "tb_attend_paged_q8", attend(most=16)) == (3, "null context")
    assert call(lib, "tb_attend_paged_q8", attend(pages(table=None)))[0] == 3
    assert call(lib, "tb_attend_paged_q8", attend(pages(requests=8193)))[0] == 3
    assert call(lib, "tb_attend_paged_q8", attend(pages(width=1 << 27)))[0] == 3
    assert call(lib, "tb_attend_paged_q8", attend(starts=None, most=1, tokens=3)) == (3, "null context")
    assert call(lib, "tb_attend_paged_q8", attend(tokens=0, q=None, out=None)) == (3, "null context")


@pytest.mark.parametrize("change", [{"logits": None}, {"out": None}, {"dtype": 3}, {"vocab": 0}, {"vocab": 1 << 31}, {"stride": 99}, {"out_stride": 99}, {"total": None},
                                    {"prompt": None}, {"history": None}, {"bias": None}, {"bias_count": None}, {"masks": 0}, {"allowed_stride": 3}, {"logits": AT + 2},
                                    {"allowed": AT + 2}, {"out_stride": 104}, {"bias_stride": 1025}, {"history_stride": 1 << 20}])
def test_bad_logits(lib, change):
    status, text = call(lib, "tb_logits_adjust", logits(**change))
    assert status == 3 and text.startswith("tb_logits_adjust")


def test_logits_without_their_parts(lib):
    assert call(lib, "tb_logits_adjust", logits(history=None, prompt=None, total=None, repetition=None, frequency=None, presence=None, bias_token=None, allowed=None)) == (3, "null context")
    assert call(lib, "tb_logits_adjust", logits(rows=0, logits=None)) == (3, "null context")
    assert call(lib, "tb_logits_adjust", logits(rows=1, stride=0, out_stride=0, masks=1)) == (3, "null context")
