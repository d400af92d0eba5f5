"""What the operators of several replies to one prompt refuse, without a GPU: sizes at the C entries (which return before any
launch), tensors and plans at the Python ones."""
import pytest
import torch

from nano_vllm_cpp_b200.csrc import ops

BAD_DTYPE, BAD_SIZE, UNSUPPORTED = -2, -3, -4


def logprobs(dt=0, stride=100, R=1, V=100, K=0, ids=None, lps=None):
    return ops.lib().nv_token_logprobs(None, dt, stride, R, V, None, None, None, None, K, ids, lps, None, None)


def test_log_probabilities_refuse_sizes():
    assert ops.lib().nv_token_logprobs_max_top() == ops.MAX_TOP_LOGPROBS
    assert logprobs(R=0) == 0
    assert logprobs(dt=2) == BAD_DTYPE
    assert logprobs(R=-1) == BAD_SIZE
    assert logprobs(V=0) == BAD_SIZE
    assert logprobs(stride=99) == BAD_SIZE
    assert logprobs(K=-1) == BAD_SIZE
    assert logprobs(K=5) == BAD_SIZE                                        # alternatives without a place for them
    assert logprobs(K=ops.MAX_TOP_LOGPROBS + 1, ids=16, lps=16) == BAD_SIZE
    assert logprobs(V=3, stride=3, K=4, ids=16, lps=16) == BAD_SIZE         # more alternatives than ids


def test_page_copies_refuse_sizes():
    call = lambda A, n, N: ops.lib().nv_copy_pages(None, A, n, None, None, None, N, None, None)
    assert call(0, 0, 5) == 0 and call(5, 64, 0) == 0
    for bad in ((-1, 0, 1), (1, 0, -1), (1, -1, 1), (70000, 64, 1), (1, 1 << 40, 1 << 30)):
        assert call(*bad) == BAD_SIZE


def shared(q_dt=1, R=1, M=0, groups=0, scale=1.0, Hq=4, Hkv=2, D=64, page=16, pages=8, own=1, ours=0):
    return ops.lib().nv_attention_decode_shared(None, q_dt, 512, None, None, 1, None, 4, None, None, None, R, None, None, None, M, None,
                                                None, None, groups, scale, None, 1, Hq, Hkv, D, page, pages, own, ours, None, None, 0, 0.0,
                                                0, 0.0, None, 0, None)


def test_shared_attention_refuses_sizes():
    assert shared(R=0) == 0
    assert shared(q_dt=2) == BAD_DTYPE
    for kw in (dict(Hq=3), dict(Hkv=0), dict(Hq=0), dict(D=60), dict(D=264), dict(D=0), dict(page=24), dict(page=0), dict(scale=0.0),
               dict(scale=-1.0), dict(scale=float("nan"))):
        assert shared(**kw) == UNSUPPORTED, kw
    for kw in (dict(R=-1), dict(M=-1), dict(groups=-1), dict(own=0), dict(ours=-1), dict(pages=0), dict()):        # (no scratch)
        assert shared(**kw) == BAD_SIZE, kw


def test_shared_prefix_packs_its_groups():
    packed, members = ops.SharedPrefix.pack([([4, 1], 32), ([2], 7)], 6)
    assert members == 3 and ops.SharedPrefix.facts([([4, 1], 32), ([2], 7)], 6) == (32, 0, 32)
    assert ops.SharedPrefix.facts([([0, 1, 2], 48), ([3], 16)], 4) == (48, 16, 96) and ops.SharedPrefix.facts([], 3) == (0, 0, 0)
    assert packed[:6] == [0, 32, 7, 0, 32, 0]                               # shared positions of every row
    assert packed[6:12] == [-1, 0, 1, -1, 0, -1]                            # its group
    assert packed[12:15] == [4, 1, 2]                                       # the groups' rows, the leading one first
    assert packed[18:21] == [0, 2, 3] and packed[21:23] == [32, 7] and packed[23:] == [4, 2]
    assert ops.SharedPrefix.pack([], 2) == ([0, 0, -1, -1, 0, 0, 0], 0)


def test_shared_prefix_packs_room_for_more_groups():
    packed, members = ops.SharedPrefix.pack([([4, 1], 32), ([2], 7)], 6, 4)
    assert members == 3 and packed[:18] == ops.SharedPrefix.pack([([4, 1], 32), ([2], 7)], 6)[0][:18]
    assert packed[18:23] == [0, 2, 3, 3, 3] and packed[23:27] == [32, 7, 0, 0] and packed[27:] == [4, 2, 0, 0]
    with pytest.raises(ops.KernelError):
        ops.SharedPrefix.pack([([4, 1], 32), ([2], 7)], 6, 1)


def test_shared_prefix_refuses_arrays_and_room_that_do_not_fit():
    groups = [([0, 1], 32)]
    buf = torch.zeros(13, dtype=torch.int32)                                # 3 rows, 1 group
    ops.SharedPrefix(groups, 3, "cpu", buf=buf)
    for kw in (dict(buf=buf[:12]), dict(buf=buf.long()), dict(room=(1, 1)), dict(room=(4, 1)), dict(room=(3, 2), buf=buf)):
        with pytest.raises(ops.KernelError):
            ops.SharedPrefix(groups, 3, "cpu", **kw)


def test_steps_of_about_the_same_prefixes_share_a_capture():
    from nano_vllm_cpp_b200.engine.runner import ModelRunner
    rounded = lambda sizes, n, rows: ModelRunner._rounded_facts([([0] * s, n) for s in sizes], rows)
    assert rounded([8], 2048, 8) == ((2048, 2048, 14336), (8, 1)) and rounded([8], 2049, 8) == ((2560, 2048, 14336), (8, 1))
    assert rounded([3, 2], 100, 6) == ((112, 0, 256), (5, 2)) and rounded([33], 64, 64)[1] == (40, 1) and rounded([33], 64, 34)[1] == (34, 1)
    for rows in range(2, 70):
        for k in range(2, rows + 1):
            members, groups = rounded([k] * 9, 16, 9 * rows)[1]
            assert 9 * k <= members <= min(9 * rows, 9 * k * 5 // 4 + 1) and groups == 10
    for n in range(1, 3000):
        longest, shortest, repeated = rounded([2], n, 2)[0]
        assert n <= longest <= n * 5 // 4 + 1 and shortest == repeated and shortest <= n <= shortest * 5 // 4 + 1


def test_sharing_is_a_matter_of_bytes_rows_and_heads():
    pays = lambda R, M, g, Hq, Hkv, repeated, dt=1, D=128, page=16: ops.lib().nv_attention_shared_pays(R, M, g, Hq, Hkv, D, page, dt, repeated)
    assert not pays(4, 0, 0, 16, 16, 0) and not pays(4, 4, 1, 16, 16, 0)
    assert pays(64, 64, 1, 28, 4, 63 * 8192) and not pays(4, 4, 1, 16, 16, 3 * 496)
    assert pays(4, 4, 1, 16, 16, 3 * 1500) and pays(4, 4, 1, 8, 2, 3 * 500, dt=0) and not pays(4, 4, 1, 16, 16, 3 * 500, dt=0)
    assert pays(128, 128, 1, 28, 4, 1 << 40)                                 # (some 10^15 bytes)


@pytest.mark.parametrize("groups", [[([], 16)], [([0], -1)], [([3], 16)], [([-1], 16)], [([0, 0], 16)], [([0], 16), ([1, 0], 16)]])
def test_shared_prefix_refuses_groups(groups):
    with pytest.raises(ops.KernelError):
        ops.SharedPrefix.pack(groups, 3)


def test_tensors_of_the_host_are_refused():
    x, i = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ops.KernelError):
        ops.token_logprobs(x, i, torch.zeros(2))
    with pytest.raises(ops.KernelError):
        ops.PageArrays([torch.zeros(4, 2, 16, 8)])
    with pytest.raises(ops.KernelError):
        ops.PageArrays([])


def test_bound_arrays_come_with_what_the_block_tables_must_cover():
    shared = ops.SharedPrefix([([0, 1], 32)], 3, "cpu", room=(3, 2))
    pack = lambda groups: torch.tensor(ops.SharedPrefix.pack(groups, 3, 2)[0], dtype=torch.int32)
    assert shared.reach == 32
    shared.bind(pack([([0, 1, 2], 4096)]), reach=4096)
    assert shared.reach == 4096
    shared.bind(pack([([2], 5)]))                                           # (not said: the kernels look)
    assert shared.reach == 0


def test_own_keys_are_cut_by_the_heads_that_a_block_takes():
    splits = lambda R, Hq, Hkv, D, ours, most, page=16: ops.lib().nv_attention_shared_own_splits(R, R, 1, Hq, Hkv, D, page, 1, ours, most)
    assert splits(40, 64, 4, 64, 0, 700) == 1                               # 320 blocks of eight heads, of 444 that live on the GPU
    assert splits(40, 64, 4, 112, 0, 700) == 2                              # 160 of 16 heads
    assert splits(44, 32, 2, 128, 4, 300) == 1 and splits(40, 28, 4, 128, 0, 700) == splits(40, 32, 4, 128, 0, 700) == 2
    # heads of 256: 88 blocks, where 24 of the shared part leave 124 multiprocessors with two each; 128 in what 128 leave, 384 keys a split
    assert splits(44, 16, 1, 256, 4, 300) == (24 + 2 * 124) // 88 == 3 and splits(64, 16, 1, 256, 16, 512) == 2
