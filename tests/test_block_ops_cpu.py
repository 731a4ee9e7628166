"""What the operators between the packed linears refuse before anything is launched, and their plans; no GPU needed."""
import ctypes
import os
import re
import subprocess

import pytest

import __graft_entry__ as entry

INVALID = 1


@pytest.fixture(scope="module")
def qi():
    module = entry.load_package()
    if not os.path.exists(module.LIB_PATH):
        module.build()
    return module


def cache(qi, **changes):
    fields = dict(k_codes=256, v_codes=512, k_scales=1024, v_scales=2048, layers=2, pages=10, page_tokens=32, kv_heads=4, head_dim=128)
    fields.update(changes)
    return qi.qi_kv_cache(**fields)


def pages(qi, **changes):
    fields = dict(table=256, lengths=512, references=1024, sequences=3, table_pages=5)
    fields.update(changes)
    return qi.qi_kv_pages(**fields)


def batch(qi, **changes):
    fields = dict(slots=256, offsets=512, entries=2, tokens=4, most=3)
    fields.update(changes)
    return qi.qi_kv_batch(**fields)


def without_a_device(status):
    """Sound arguments get as far as the launch, which has no device here. (Where there is one, made-up addresses must not be launched.)"""
    return status not in (0, INVALID)


def test_sound_arguments_reach_the_launch(qi):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    for status in every_call(qi, cache(qi), pages(qi), batch(qi)):
        assert without_a_device(status)
    library, c, p = qi.lib(), ctypes.byref(cache(qi)), ctypes.byref(pages(qi))
    assert without_a_device(library.qi_kv_pages_reserve_ex(c, p, 256, 512, 1, 768, 256, 1 << 20, None))
    assert without_a_device(library.qi_kv_pages_fork_ex(c, p, 256, 512, 1, 768, 256, 1 << 20, None))
    assert without_a_device(library.qi_kv_pages_free_ex(c, p, 256, 1, None))
    assert without_a_device(library.qi_kv_pages_compact_ex(c, p, 256, 256, 1 << 20, None))
    assert without_a_device(library.qi_kv_pages_copy_ex(c, 256, 512, 1, None))
    assert without_a_device(library.qi_gated_norm_ex(ctypes.byref(norm_call(qi)), None))


def norm_call(qi, **changes):
    fields = dict(rows=4, width=64, kind=qi.NORM_RMS, epsilon=1e-6, residual=256, residual_dtype=0, branch=512, branch_dtype=1, branch_norm=1, branch_weight=1024, residual_scale=1.0, gate=2048,
                  scale=0, shift=0, vector_dtype=1, ld_vector=64, rows_per_vector=4, weight=4096, residual_out=256, y=512, y_dtype=1)
    fields.update(changes)
    return qi.qi_gated_norm(**fields)


BAD_CACHES = [dict(k_codes=0), dict(v_codes=264), dict(k_scales=0), dict(v_scales=2), dict(layers=0), dict(pages=0), dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=512),
              dict(kv_heads=0), dict(head_dim=96), dict(head_dim=256)]
BAD_PAGES = [dict(table=0), dict(lengths=0), dict(references=0), dict(references=2), dict(sequences=0), dict(table_pages=0), dict(table_pages=(1 << 19) + 1)]
BAD_BATCHES = [dict(offsets=0), dict(offsets=2), dict(entries=-1), dict(entries=65536), dict(tokens=-1), dict(most=-1)]


def every_call(qi, c, p, b):
    """The calls that take all three, with sound arguments otherwise."""
    library, ref = qi.lib(), ctypes.byref
    call = qi.qi_kv_attention(layer=1, heads=8, q=256, ld_q=1024, y=512, ld_y=1024, lse=0, scale=0.1, causal=1, window=0, max_length=100)
    yield library.qi_kv_append_ex(ref(c), ref(p), ref(b), 1, 256, 512, qi.DTYPE_F16, 512, 512, None)
    yield library.qi_kv_read_ex(ref(c), ref(p), ref(b), 1, 256, 512, qi.DTYPE_F32, 512, 512, None)
    yield library.qi_kv_attention_ex(ref(c), ref(p), ref(b), ref(call), 256, 1 << 30, None)


@pytest.mark.parametrize("changes", BAD_CACHES, ids=str)
def test_unfit_caches(qi, changes):
    for status in every_call(qi, cache(qi, **changes), pages(qi), batch(qi)):
        assert status == INVALID
    library, c, size = qi.lib(), cache(qi, **changes), ctypes.c_size_t(0)
    assert library.qi_kv_pages_workspace(ctypes.byref(c), ctypes.byref(pages(qi)), ctypes.byref(size)) == INVALID
    assert library.qi_kv_pages_copy_ex(ctypes.byref(c), 256, 512, 1, None) == INVALID
    assert library.qi_kv_pages_free_ex(ctypes.byref(c), ctypes.byref(pages(qi)), 256, 1, None) == INVALID


@pytest.mark.parametrize("changes", BAD_PAGES, ids=str)
def test_unfit_tables(qi, changes):
    for status in every_call(qi, cache(qi), pages(qi, **changes), batch(qi)):
        assert status == INVALID


@pytest.mark.parametrize("changes", BAD_BATCHES, ids=str)
def test_unfit_batches(qi, changes):
    for status in every_call(qi, cache(qi), pages(qi), batch(qi, **changes)):
        assert status == INVALID


def test_unfit_arguments_of_the_cache(qi):
    library, c, p, b = qi.lib(), ctypes.byref(cache(qi)), ctypes.byref(pages(qi)), ctypes.byref(batch(qi))
    for call in (library.qi_kv_append_ex, library.qi_kv_read_ex):
        assert call(c, p, b, -1, 256, 512, qi.DTYPE_F16, 512, 512, None) == INVALID
        assert call(c, p, b, 2, 256, 512, qi.DTYPE_F16, 512, 512, None) == INVALID
        assert call(c, p, b, 0, 0, 512, qi.DTYPE_F16, 512, 512, None) == INVALID
        assert call(c, p, b, 0, 256, 520, qi.DTYPE_F16, 512, 512, None) == INVALID
        assert call(c, p, b, 0, 256, 512, 2, 512, 512, None) == INVALID
        assert call(c, p, b, 0, 256, 512, qi.DTYPE_F16, 511, 512, None) == INVALID
        assert call(c, p, b, 0, 256, 512, qi.DTYPE_F16, 512, 516, None) == INVALID
        assert call(c, p, b, 0, 256, 512, qi.DTYPE_F32, 514, 512, None) == INVALID
        assert call(None, p, b, 0, 256, 512, qi.DTYPE_F32, 512, 512, None) == INVALID
        # an empty batch is no call at all
        assert call(c, p, ctypes.byref(batch(qi, entries=0)), 0, 256, 512, qi.DTYPE_F32, 512, 512, None) == 0
        assert call(c, p, ctypes.byref(batch(qi, most=0, tokens=0)), 0, 256, 512, qi.DTYPE_F32, 512, 512, None) == 0


@pytest.mark.parametrize("kv_heads", [1, 4, 64, 4096])
def test_any_bound_of_new_tokens_is_cut_to_what_a_table_holds(qi, kv_heads):
    # 5 pages of 32 tokens: 10 blocks a head, whatever `most` says; units of blocks that no sequence can have overflowed their token numbers
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    library, c, p, width = qi.lib(), cache(qi, kv_heads=kv_heads), pages(qi), kv_heads * 128
    for most in (160, 161, 1 << 20, 0x7fffffff - 30, 0x7fffffff):
        b = batch(qi, most=most)
        for call in (library.qi_kv_append_ex, library.qi_kv_read_ex):
            assert without_a_device(call(ctypes.byref(c), ctypes.byref(p), ctypes.byref(b), 1, 256, 512, qi.DTYPE_F16, width, width, None))


@pytest.mark.parametrize("changes", [dict(layer=2), dict(layer=-1), dict(heads=0), dict(heads=6), dict(heads=-4), dict(heads=4 << 20), dict(q=0), dict(q=264), dict(y=0), dict(y=8), dict(lse=2), dict(ld_q=1016),
                                     dict(ld_y=1020), dict(ld_q=1028), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1),
                                     dict(max_length=-1)], ids=str)
def test_unfit_attention(qi, changes):
    fields = dict(layer=1, heads=8, q=256, ld_q=1024, y=512, ld_y=1024, lse=0, scale=0.1, causal=1, window=0, max_length=100)
    fields.update(changes)
    call = qi.qi_kv_attention(**fields)
    assert qi.lib().qi_kv_attention_ex(ctypes.byref(cache(qi)), ctypes.byref(pages(qi)), ctypes.byref(batch(qi)), ctypes.byref(call), 256, 1 << 40, None) == INVALID


def test_attention_refuses_a_workspace_that_is_too_small(qi):
    library, c, p, size = qi.lib(), cache(qi), pages(qi), ctypes.c_size_t(0)
    b = batch(qi, entries=1, tokens=1, most=1)
    assert library.qi_kv_attention_workspace(ctypes.byref(c), ctypes.byref(b), 8, 5000, ctypes.byref(size)) == 0 and size.value > 0
    call = qi.qi_kv_attention(layer=1, heads=8, q=256, ld_q=1024, y=512, ld_y=1024, lse=0, scale=0.1, causal=1, window=0, max_length=5000)
    for workspace, count in ((256, size.value - 1), (0, size.value), (264, size.value)):
        assert library.qi_kv_attention_ex(ctypes.byref(c), ctypes.byref(p), ctypes.byref(b), ctypes.byref(call), workspace, count, None) == INVALID
    # any window fits what is asked for without one
    for window in (1, 77, 900, 4999, 5000, 1 << 30):
        if pytest.importorskip("torch").cuda.is_available():
            break
        call.window = window
        assert without_a_device(library.qi_kv_attention_ex(ctypes.byref(c), ctypes.byref(p), ctypes.byref(b), ctypes.byref(call), 256, size.value, None))


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("kv_heads,heads", [(4, 32), (1, 1), (8, 24), (32, 32), (80, 80), (2, 40)])
def test_a_workspace_for_the_largest_batch_serves_the_smaller_ones(qi, kv_heads, heads, head_dim):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    library, c, p = qi.lib(), cache(qi, kv_heads=kv_heads, head_dim=head_dim), pages(qi, table_pages=400)
    size, width = ctypes.c_size_t(0), heads * head_dim
    for entries, most, length in ((8, 4096, 8192), (70, 12, 5000), (3, 300, 700), (64, 1, 8192), (1, 40, 12800), (5, 2, 128)):
        assert library.qi_kv_attention_workspace(ctypes.byref(c), ctypes.byref(batch(qi, entries=entries, tokens=entries * most, most=most)), heads, length, ctypes.byref(size)) == 0
        bound = size.value
        for fewer in sorted({1, 2, 7, entries // 2, entries - 1, entries}):
            for less in sorted({0, 1, 2, 3, 9, 17, 100, most // 2, most - 1, most}):
                for shorter, window in ((length, 0), (length // 3, 0), (100, 0), (length, 50), (length, 1000)):
                    if not (0 < fewer <= entries and 0 <= less <= most):
                        continue
                    b = batch(qi, entries=fewer, tokens=fewer * less, most=less)
                    assert library.qi_kv_attention_workspace(ctypes.byref(c), ctypes.byref(b), heads, shorter, ctypes.byref(size)) == 0 and size.value <= bound
                    call = qi.qi_kv_attention(layer=1, heads=heads, q=256, ld_q=width, y=512, ld_y=width, lse=0, scale=0.1, causal=1, window=window, max_length=shorter)
                    status = library.qi_kv_attention_ex(ctypes.byref(c), ctypes.byref(p), ctypes.byref(b), ctypes.byref(call), 256, bound, None)
                    assert status != INVALID, (fewer, less, shorter, window)


def test_unfit_page_lists(qi):
    library, c, p = qi.lib(), ctypes.byref(cache(qi)), ctypes.byref(pages(qi))
    size = ctypes.c_size_t(0)
    assert library.qi_kv_pages_workspace(c, p, ctypes.byref(size)) == 0
    # counters, two lists, where each page went, a snapshot of the tables and lengths
    assert size.value == 4 * (4 + 10 + 10 + 10 + 15 + 3)
    for call in (library.qi_kv_pages_reserve_ex, library.qi_kv_pages_fork_ex):
        assert call(c, p, 0, 512, 1, 768, 256, size.value, None) == INVALID
        assert call(c, p, 256, 0, 1, 768, 256, size.value, None) == INVALID
        assert call(c, p, 256, 512, 1, 0, 256, size.value, None) == INVALID
        assert call(c, p, 256, 512, 4, 768, 256, size.value, None) == INVALID  # more than there are sequences
        assert call(c, p, 256, 512, -1, 768, 256, size.value, None) == INVALID
        assert call(c, p, 256, 512, 1, 768, 256, size.value - 1, None) == INVALID
        assert call(c, p, 256, 512, 1, 768, 0, size.value, None) == INVALID
    assert library.qi_kv_pages_compact_ex(c, p, 256, 256, size.value - 1, None) == INVALID
    assert library.qi_kv_pages_compact_ex(c, p, 0, 256, size.value, None) == INVALID
    assert library.qi_kv_pages_free_ex(c, p, 0, 1, None) == INVALID
    assert library.qi_kv_pages_free_ex(c, p, 256, 0, None) == 0
    assert library.qi_kv_pages_copy_ex(c, 256, 0, 1, None) == INVALID
    assert library.qi_kv_pages_copy_ex(c, 256, 512, 11, None) == INVALID


@pytest.mark.parametrize("changes", [dict(rows=-1), dict(width=0), dict(width=12), dict(width=16392), dict(kind=2), dict(residual=0), dict(residual=264), dict(residual_dtype=2), dict(branch_dtype=-1),
                                     dict(y=0, residual_out=0), dict(epsilon=-1.0), dict(epsilon=float("nan")), dict(branch=0), dict(ld_vector=56), dict(ld_vector=68),
                                     dict(rows_per_vector=0), dict(gate=8), dict(weight=4), dict(y_dtype=3), dict(vector_dtype=7)], ids=str)
def test_unfit_norms(qi, changes):
    assert qi.lib().qi_gated_norm_ex(ctypes.byref(norm_call(qi, **changes)), None) == INVALID
    assert qi.lib().qi_gated_norm_ex(None, None) == INVALID


def test_structures_that_do_not_belong_together(qi):
    torch = pytest.importorskip("torch")
    codes, scales = torch.zeros(1, 4, 2, 32, 64, dtype=torch.uint8), torch.zeros(1, 4, 2, 2)
    qi.KvCache(codes, codes, scales, scales)
    with pytest.raises(ValueError):
        qi.KvCache(codes, codes[:, :3], scales, scales)
    with pytest.raises(ValueError):
        qi.KvCache(codes, codes, scales, scales[..., :1])
    with pytest.raises(ValueError):
        qi.KvPages(torch.zeros(3, 5, dtype=torch.int32).T, torch.zeros(5, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))


def test_structures_of_other_types_and_sizes(qi):
    # what the device cannot see: int64 read as int32 pairs, scales of half the size written beyond, references shorter than the pool
    torch = pytest.importorskip("torch")
    codes, scales = torch.zeros(1, 4, 2, 32, 64, dtype=torch.uint8), torch.zeros(1, 4, 2, 2)
    for k, v, ks, vs in ((codes.float(), codes, scales, scales), (codes.view(torch.int8), codes, scales, scales), (codes, codes.char(), scales, scales), (codes, codes, scales.half(), scales),
                         (codes, codes, scales, scales.double()), (codes, codes, scales, scales.int()), (codes.to("meta"), codes, scales, scales), (codes, codes, scales, scales.to("meta"))):
        with pytest.raises(ValueError):
            qi.KvCache(k, v, ks, vs)
    table, lengths, references = torch.zeros(3, 5, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    for parts in ((table.long(), lengths, references), (table, lengths.long(), references), (table, lengths, references.long()), (table.float(), lengths, references),
                  (table, lengths, torch.zeros(8, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError):
            qi.KvPages(*parts)
    offsets, slots = torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for parts in ((slots, offsets.long()), (slots.long(), offsets), (slots[:2], offsets), (None, offsets[:0]), (None, offsets.float()), (torch.zeros(6, dtype=torch.int32)[::2], offsets)):
        with pytest.raises(ValueError):
            qi.KvBatch(*parts, 5, 2)
    for word in (torch.zeros(1), torch.zeros(1, dtype=torch.int64), torch.zeros(0, dtype=torch.int32)):
        with pytest.raises(ValueError):
            qi.KvBatch(slots, offsets, 5, 2, word)
    for status in every_call(qi, cache(qi), pages(qi), batch(qi, shortage=258)):
        assert status == INVALID
    qi.KvBatch(None, offsets, 5, 2), qi.KvBatch(slots, offsets, 5, 2), qi.KvBatch(torch.zeros(9, dtype=torch.int32), offsets, 5, 2)


def test_lists_and_pools_that_are_too_short(qi):
    torch = pytest.importorskip("torch")
    ints = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    cache_ = qi.KvCache(torch.zeros(1, 4, 2, 32, 64, dtype=torch.uint8), torch.zeros(1, 4, 2, 32, 64, dtype=torch.uint8), torch.zeros(1, 4, 2, 2), torch.zeros(1, 4, 2, 2))
    pages_, batch_ = qi.KvPages(torch.zeros(3, 5, dtype=torch.int32), ints(3), ints(4)), qi.KvBatch(None, ints(3), 4, 2)
    few = qi.KvPages(torch.zeros(3, 5, dtype=torch.int32), ints(3), ints(3))  # a reference less than pages
    elsewhere = [qi.KvPages(*(t.to("meta") if i == part else t for i, t in enumerate((torch.zeros(3, 5, dtype=torch.int32), ints(3), ints(4))))) for part in range(3)]
    work = torch.zeros(1 << 12, dtype=torch.uint8)
    calls = [lambda p, l: qi.kv_pages_reserve_ex(cache_, p, l, ints(3), 3, ints(1), work), lambda p, l: qi.kv_pages_reserve_ex(cache_, p, ints(3), l, 3, ints(1), work),
             lambda p, l: qi.kv_pages_fork_ex(cache_, p, l, ints(3), 3, ints(1), work), lambda p, l: qi.kv_pages_fork_ex(cache_, p, ints(3), l, 3, ints(1), work),
             lambda p, l: qi.kv_pages_free_ex(cache_, p, l, 3)]
    for call in calls:
        for bad in (ints(2), ints(3).long(), ints(6)[::2], torch.zeros(3), ints(3).to("meta")):
            with pytest.raises(ValueError):
                call(pages_, bad)
        for unfit in [few] + elsewhere:
            with pytest.raises(ValueError):
                call(unfit, ints(3))
    copies = [lambda l: qi.kv_pages_copy_ex(cache_, l, ints(3), 3), lambda l: qi.kv_pages_copy_ex(cache_, ints(3), l, 3)]
    for call in copies:
        for bad in (ints(2), ints(3).long()):
            with pytest.raises(ValueError):
                call(bad)
    for word in (ints(0), ints(1).long()):
        with pytest.raises(ValueError):
            qi.kv_pages_compact_ex(cache_, pages_, word, work)
        with pytest.raises(ValueError):
            qi.kv_pages_reserve_ex(cache_, pages_, ints(3), ints(3), 3, word, work)
    x = torch.zeros(4, 2, 64, dtype=torch.float16)
    for call in (lambda: qi.kv_append_ex(cache_, few, batch_, 0, x, x, qi.DTYPE_F16, 128, 128), lambda: qi.kv_read_ex(cache_, few, batch_, 0, x, x, qi.DTYPE_F16, 128, 128),
                 lambda: qi.kv_attention_ex(cache_, few, batch_, 0, x, 128, x, 128, 2, 1.0, 160, workspace=work), lambda: qi.kv_pages_compact_ex(cache_, few, ints(1), work),
                 lambda: qi.kv_append_ex(cache_, pages_, qi.KvBatch(None, ints(3).to("meta"), 4, 2), 0, x, x, qi.DTYPE_F16, 128, 128),
                 lambda: qi.kv_attention_ex(cache_, pages_, qi.KvBatch(ints(2).to("meta"), ints(3), 4, 2), 0, x, 128, x, 128, 2, 1.0, 160, workspace=work)):
        with pytest.raises(ValueError):
            call()


def test_quotients_that_need_64_bits(tmp_path):
    # the kernel's own function, compiled for the host: which CTA has a round when there are more rounds than 32 bits count
    source = open(os.path.join(entry.PACKAGE_DIR, "csrc", "kv_decode.cuh"), encoding="utf-8").read()
    body = re.search(r"__device__ __forceinline__ (long long divide\(.*?\n}\n)", source, re.S).group(1)
    pairs = [(a, b) for a in (0, 1, 295, 296, 2 ** 31, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 5, 2 ** 40 + 7) for b in (1, 3, 296, 2 ** 31, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 2, 3 * 2 ** 33)]
    checks = "".join(f"if (divide({a}LL, {b}LL) != {a // b}LL) return {i + 1};" for i, (a, b) in enumerate(pairs))
    program = tmp_path / "divide.cpp"
    program.write_text("#include <cstdint>\nstatic " + body + "int main() { " + checks + " return 0; }\n")
    subprocess.run(["g++", "-std=c++17", "-o", str(tmp_path / "divide"), str(program)], check=True)
    assert subprocess.run([str(tmp_path / "divide")]).returncode == 0
