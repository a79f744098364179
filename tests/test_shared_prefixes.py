"""The host side of shared prefixes: the description the kernels read, the cuts of the keys, what is refused, and the
refusals of the copies inside the cache."""
import numpy as np
import pytest

from zinfer_b200 import kernels as k


def described(groups, n):
    words = np.full(k.SharedPrefixes.word_count(n), 77, dtype=np.int32)
    return words, k.SharedPrefixes.fill(words, groups, n)


def test_words_name_rows_keys_and_first_own_keys():
    words, kept = described([((4, 1), 130), ((0,), 64), ((2, 5, 3), 64), ((6, 7), 0)], 8)
    assert kept == ((2, 130), (3, 64))                       # a row alone and a group without keys share nothing
    assert words[0] == 2 and words[4:20].tolist() == [0, 2, 130, 4, 2, 3, 64, 2] + [0] * 8
    assert words[20:28].tolist() == [4, 1, 2, 5, 3, 0, 0, 0]
    assert words[28:].tolist() == [0, 130, 64, 64, 130, 64, 0, 0]


def test_a_batch_without_groups():
    for n in (1, 2, 3):
        words, kept = described([], n)
        assert kept == () and not words.any()


def test_every_row_in_one_group_and_the_largest_number_of_groups():
    for n in (10, 11):
        words, kept = described([((2 * i, 2 * i + 1), i + 1) for i in range(5)], n)
        assert len(kept) == 5 and words[4:24].reshape(5, 4).tolist() == [[2 * i, 2, i + 1, 2 * i] for i in range(5)]
        assert words[24 + n:34 + n].tolist() == [1, 1, 2, 2, 3, 3, 4, 4, 5, 5]


@pytest.mark.parametrize("groups", [[((0, 0), 5)], [((0, 1), 5), ((1, 2), 5)], [((0, 4), 5)], [((-1, 0), 5)], [((0, 1), -1)],
                                    [((0, 1), 1 << 30)], [((0,), 5), ((0, 1), 5)]])
def test_groups_that_are_refused(groups):
    with pytest.raises(k.KernelError):
        described(groups, 4)


@pytest.mark.parametrize("sms", [1, 148])
@pytest.mark.parametrize("groups,n", [((), 1), (((2, 1),), 2), (((64, 8192),), 64), (((9, 300), (9, 6000), (9, 547)), 40),
                                      (((2, 32768),), 3), (((128, 100000),), 128)])
def test_layouts_reach_every_key(groups, n, sms):
    """Tasks for every tile and chunk of every group, splits for the longest prefix, own chunks up to the longest row's end."""
    for G, n_kv, rows in ((1, 8, 16), (4, 8, 128), (16, 1, 32), (3, 5, 16)):
        for own, fma in ((1, False), (127, True), (128, False), (129, False), (5000, True), (5000, False)):
            chunk, tasks, splits, own_splits, own_keys = k.shared_layout(groups, n, G, n_kv, rows, own, sms, fma)
            assert chunk % 64 == 0 and own_keys % 64 == 0 and own_splits >= 1
            assert own_splits * own_keys >= own
            assert tasks >= sum(-(-r * G // rows) * -(-keys // chunk) for r, keys in groups)
            assert all(splits * chunk >= keys for _, keys in groups)
            assert (splits > 0) == bool(groups)


def test_layouts_of_many_long_groups_are_quick_and_even():
    """Blocks of some lengths for groups that are more than the SMs, and a second wave where one would leave SMs idle."""
    import time
    begin = time.perf_counter()
    k.shared_layout(((2, 1 << 20),) * 300, 600, 4, 8, 128, 5, 148)
    k.shared_layout(((2, (1 << 30) - 1),) * 3, 6, 4, 8, 16, 5, 148)
    assert time.perf_counter() - begin < 1.0
    chunk, tasks, *_ = k.shared_layout(((6, 16384),) * 12, 72, 4, 8, 128, 1, 148)
    assert 148 < 8 * tasks <= 296 and chunk < 16384 // 2


def test_descriptions_with_one_key_have_the_same_launches():
    for groups, like in ((((8, 4096),), ((8, 4090),)), (((3, 700), (2, 100)), ((3, 641), (2, 128)))):
        a, b = (k.SharedPrefixes([(list(range(10 * g, 10 * g + rows)), keys) for g, (rows, keys) in enumerate(gs)], 24, "cpu")
                for gs in (groups, like))
        for own, own_like in ((5, 128), (129, 192)):
            assert a.key(own) == b.key(own_like)
            for geometry in ((4, 8, 128), (1, 8, 16), (16, 1, 32)):
                assert a.layout(*geometry, own, 148) == b.layout(*geometry, own_like, 148)
        assert a.key(128) != b.key(129)
    with pytest.raises(k.KernelError):
        k.SharedPrefixes([], 4, "cpu", words=a.words)


def test_a_layout_changes_seldom_while_sequences_grow():
    seen = {k.shared_layout(((8, 4096),), 8, 4, 8, 128, own, 148) for own in range(1, 4097)}
    assert len(seen) <= 11


@pytest.mark.parametrize("src,dst,count", [([0, 1], [2], None), ([0], [0], None), ([0, 1], [2, 2], None), ([0, 2], [2, 3], None),
                                           ([0], [4], None), ([-1], [1], None), ([4], [1], None), ([0], [-1], None), ([0], [1], [17]),
                                           ([0], [1], [-1]), ([0], [1], [1, 2]), ([1 << 32], [1], None), ([3, 3, 1], [0, 2, 3], None)])
@pytest.mark.parametrize("kind", [list, np.array])
def test_moves_that_are_refused(src, dst, count, kind):
    with pytest.raises(k.KernelError):
        k._moves(kind(src), kind(dst), count if count is None else kind(count), 4, 16, "copy")


def test_moves_that_are_taken():
    src, dst, count = k._moves([0, 0, 3], np.array([1, 2, 4]), [0, 16, 5], 5, 16, "copy")
    assert src[1] == dst[1] == count[1] == 3 and list(src[2]) == [0, 0, 3] and dst[2].dtype == np.int32
    assert k._moves([], [], None, 4, 1, "copy")[0][1] == 0
    n = 3000
    k._moves(list(range(n)), list(range(n, 2 * n))[::-1], None, 2 * n, 1, "copy")
    with pytest.raises(k.KernelError):
        k._moves(list(range(n)), [*range(n, 2 * n - 1), 17], None, 2 * n, 1, "copy")


@pytest.mark.parametrize("views", [(0, 1, 1, 1, 1, 4, 1, 4), (64, 1, 1, 1, 0, 4, 1, 4), (64, 1, 1, 1, 1, 3, 1, 4), (64, 1, 1, 1, 1, 4, 0, 4),
                                   (64, 1, 1, 1, 1, 4, 1, 0)])
def test_the_launcher_refuses_what_it_cannot_copy(views):
    """No address, no layers, too few entries for the moves, no heads, nothing in a unit: before anything is launched."""
    src, dst, _ = k._moves([0], [3], None, 4, 1, "copy")
    desc = np.array(views, dtype=np.int64)
    assert k._fn("cache_copy", "zk_cache_copy")(desc.ctypes.data, 1, src[0], dst[0], None, 1, 1, None) == -22


@pytest.mark.parametrize("head_dim,value_dim,scale,takes", [
    (256, None, None, True), (257, None, None, False), (640, None, None, False), (64, 257, None, False), (320, 64, None, False),
    (64, None, 0.0, False), (64, None, -0.125, False), (64, None, float("inf"), False), (64, None, float("nan"), False), (64, 256, 2.0, True)])
def test_attention_takes_prefixes_where_the_kernels_do(head_dim, value_dim, scale, takes):
    """The layer's rule and the kernels' refusals are one: a step never meets sizes that its kernel turns down."""
    from zinfer_b200.parts.attention import GqaAttention
    layer = GqaAttention(64, 4, 2, head_dim, "q", "k", "v", "o", value_dim=value_dim, scale=scale)
    assert layer.takes_prefixes is takes
    assert k.attention_shared_takes(layer.run_head_dim, layer.run_value_dim, layer.scale) is takes


@pytest.mark.parametrize("heads,n_kv,width,page,answers,keys,shares", [
    (32, 8, 32, 64, 64, 2112, False), (8, 8, 32, 64, 64, 8192, False),             # heads of 32: their own kernel is the faster
    (32, 8, 96, 64, 2, 131136, False), (32, 8, 96, 64, 9, 16448, False), (32, 8, 96, 64, 17, 8256, True), (32, 8, 96, 64, 64, 576, False),
    (6, 2, 96, 64, 13, 11008, False), (6, 2, 96, 64, 17, 8256, True), (6, 2, 96, 64, 9, 4160, False),
    (16, 8, 96, 64, 2, 131136, True), (8, 8, 96, 64, 9, 16448, True), (8, 8, 96, 64, 9, 4160, False), (16, 8, 64, 32, 9, 16448, True),
    (32, 8, 80, 64, 2, 4160, True), (32, 8, 64, 16, 5, 1088, True), (4, 4, 256, 64, 9, 576, True),     # no kernel of their own
    (32, 8, 64, 64, 5, 1088, True), (8, 8, 128, 64, 2, 4160, True)])                                   # the tensor cores
def test_bfloat16_heads_share_where_that_is_the_faster(heads, n_kv, width, page, answers, keys, shares):
    """By the kernel that would otherwise run: times of both are at the rule."""
    from types import SimpleNamespace

    import torch
    from zinfer_b200.parts.attention import GqaAttention
    layer = GqaAttention(64, heads, n_kv, width, "q", "k", "v", "o")
    ctx = SimpleNamespace(prefixes=k.SharedPrefixes([(range(answers), keys)], answers + 1, "cpu"))
    kv = SimpleNamespace(page_size=page)
    assert layer._shares(ctx, kv, torch.bfloat16) is shares
    assert layer._shares(ctx, kv, torch.float32) is True
    assert layer._shares(SimpleNamespace(prefixes=None), kv, torch.bfloat16) is False


def test_the_tensor_cores_take_what_they_take_without_shared_prefixes():
    """A fork's weights have as many bits as those of a sequence on its own."""
    import torch
    for dtype in (torch.bfloat16, torch.float32):
        for heads, n_kv in ((16, 8), (16, 1), (17, 1), (32, 2), (34, 2), (64, 1)):
            for width in (32, 64, 96, 128):
                for page in (16, 64, 192):
                    alone = dtype == torch.bfloat16 and bool(k._fn("attention_decode_tc", "zk_attn_decode_tc_takes")(heads, n_kv, width, page))
                    assert k.attention_shared_tensor_cores(dtype, heads // n_kv, width, width, page) == alone
                    code = k.dtype_code(dtype)
                    tile = k._fn("attention_shared", "zk_attn_shared_tile_rows")(code, heads // n_kv, width, width, page, 200, 9000)
                    assert tile == (128 if alone else 32)


def test_a_status_word_of_another_device_is_refused(monkeypatch):
    """A kernel would write through an address that is none on its own device."""
    import torch
    word = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(k.KernelError, match="CUDA"):
        k._need_status(word, torch.device("cuda", 0))
    monkeypatch.setattr(k, "_need", lambda *args, **kw: None)          # from here on the CPU stands for a second device
    k._need_status(word, torch.device("cpu"))
    for bad, device in ((word, torch.device("cuda", 0)), (word[:0], torch.device("cpu"))):
        with pytest.raises(k.KernelError, match="expected one"):
            k._need_status(bad, device)


def test_every_code_of_the_shared_kernel_has_a_text_that_names_it():
    """A wait that gives up, a short row, a missing page: what the engine raises says where it may have come from."""
    import re
    from pathlib import Path

    from zinfer_b200.engine.engine import _STATUS_TEXT
    source = (Path(k.__file__).parent / "csrc" / "attention_shared.cu").read_text()
    waits = {int(c) for c in re.findall(r"wait\(&?\w+(?:\[[^\]]*\])?, [^;\n]*?, (\d+)\)", source)}
    assert waits == {13, 14, 15, 16, 17, 18}
    assert all("shared prefix" in _STATUS_TEXT[c] for c in waits)
    assert {int(c) for c in re.findall(r"atomicExch\(a\.status, (\d+)\)", source)} == {2, 20} <= set(_STATUS_TEXT)
