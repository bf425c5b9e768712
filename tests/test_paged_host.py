"""The paged KV cache's operators on the CPU host: what the library and the Python entry points refuse
before anything is launched, and the test oracle of the page plan against itself."""
import pytest
import torch

from _paged import release, reserve
from modelcore_amd import _ext
from modelcore_amd.kernels.flash_attn import flash_attn
from modelcore_amd.kernels.paged import check_page_size, paged_release, paged_reserve
from modelcore_amd.kernels.qk_epilogue import check_pages, rope_norm_scale_append_paged

FAKE = 1 << 20  # never dereferenced: the checks fail first


def attention(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, kp=FAKE, vp=FAKE, table=FAKE, table_stride=8, seqlens=FAKE, cu=FAKE,
             out=FAKE, n_rows=2, total=7, longest=5, H=8, H_kv=2, D=128, n_pages=20, page=16,
             page_stride=16 * 2 * 128, max_pages=8, window=-1, dtype=_ext.BF16, scratch=None, nbytes=0)
    a.update(kw)
    if "page_stride" not in kw:
        a["page_stride"] = a["page"] * a["H_kv"] * a["D"]
    return _ext.lib().mcamd_flash_attn_paged_with_kvcache(
        a["q"], a["k"], a["v"], a["kp"], a["vp"], a["table"], a["table_stride"], a["seqlens"], a["cu"],
        a["out"], a["n_rows"], a["total"], a["longest"], a["H"], a["H_kv"], a["D"], a["n_pages"],
        a["page"], a["page_stride"], a["max_pages"], a["window"], 1, a["dtype"], a["scratch"],
        a["nbytes"], None)


@pytest.mark.parametrize("kw,code,words", [
    (dict(k=None), _ext.EINVAL, b"both k and v"),
    (dict(page=24), _ext.EINVAL, b"power of two"),
    (dict(page=8), _ext.EINVAL, b"power of two"),
    (dict(page_stride=16 * 2 * 128 - 8), _ext.EINVAL, b"page_stride"),
    (dict(page_stride=16 * 2 * 128 + 4), _ext.EINVAL, b"aligned"),
    (dict(table_stride=7), _ext.EINVAL, b"table_stride"),
    (dict(n_pages=0), _ext.EINVAL, b"empty"),
    (dict(max_pages=0), _ext.EINVAL, b"empty"),
    (dict(longest=-1), _ext.EINVAL, b"max_seqlen"),
    (dict(n_pages=1 << 28), _ext.EUNSUPPORTED, b"32-bit"),
    (dict(max_pages=1 << 27, table_stride=1 << 27), _ext.EUNSUPPORTED, b"32-bit"),
    (dict(n_rows=70000), _ext.EUNSUPPORTED, b"32-bit"),
    (dict(total=1 << 28), _ext.EUNSUPPORTED, b"32-bit"),
    (dict(cu=None), _ext.EINVAL, b"cu_seqlens"),
    (dict(dtype=3), _ext.EINVAL, b"dtype"),
    (dict(H=9), _ext.EINVAL, b"multiple"),
    (dict(H=0), _ext.EINVAL, b"positive"),
    (dict(total=-1), _ext.EINVAL, b"positive"),
    (dict(D=264), _ext.EUNSUPPORTED, b"at most 256"),
    (dict(D=12), _ext.EUNSUPPORTED, b"multiple of 16"),
    (dict(D=6, dtype=_ext.F32), _ext.EUNSUPPORTED, b"multiple of 16"),
    (dict(H=130), _ext.EUNSUPPORTED, b"64 query heads"),
    (dict(q=FAKE + 8), _ext.EINVAL, b"aligned"),
    (dict(vp=FAKE + 2), _ext.EINVAL, b"aligned"),
    (dict(k=FAKE + 4), _ext.EINVAL, b"aligned"),
    (dict(scratch=FAKE + 8, nbytes=1 << 30), _ext.EINVAL, b"aligned"),
    (dict(table=None), _ext.EINVAL, b"null"),
    (dict(seqlens=None), _ext.EINVAL, b"null"),
    (dict(out=None), _ext.EINVAL, b"null"),
])
def test_attention_refuses(kw, code, words):
    assert attention(**kw) == code
    assert words in _ext.lib().mcamd_last_error(), _ext.lib().mcamd_last_error()


def test_attention_of_nothing_is_no_launch():
    assert attention(n_rows=0, total=0) == _ext.OK
    assert attention(total=0) == _ext.OK
    assert attention(longest=0, cu=None, total=0) == _ext.OK


def test_reserve_and_release_refuse():
    lib = _ext.lib()

    def reserve_c(n_rows=2, max_pages=8, n_pages=20, page=16, total=5, stride=8, table=FAKE, count=FAKE,
                  slots=FAKE):
        return lib.mcamd_paged_reserve(table, stride, FAKE, FAKE, FAKE, count, FAKE, FAKE, slots, FAKE, FAKE,
                                       n_rows, max_pages, n_pages, page, total, None)

    def release_c(n_rows=2, max_pages=8, n_pages=20, page=16, m=1, stride=8, table=FAKE):
        return lib.mcamd_paged_release(table, stride, FAKE, FAKE, m, n_rows, FAKE, FAKE, max_pages, n_pages,
                                       page, None)

    for kw, code, words in ((dict(page=17), _ext.EINVAL, b"power of two"),
                            (dict(page=0), _ext.EINVAL, b"power of two"),
                            (dict(n_rows=-1), _ext.EINVAL, b"positive"),
                            (dict(max_pages=0), _ext.EINVAL, b"positive"),
                            (dict(stride=7), _ext.EINVAL, b"table_stride"),
                            (dict(n_pages=1 << 28), _ext.EUNSUPPORTED, b"31 bits"),
                            (dict(max_pages=1 << 28, stride=1 << 28), _ext.EUNSUPPORTED, b"31 bits"),
                            (dict(n_rows=0x7fffffff), _ext.EUNSUPPORTED, b"31 bits"),
                            (dict(table=None), _ext.EINVAL, b"null")):
        assert reserve_c(**kw) == code and words in lib.mcamd_last_error(), (kw, lib.mcamd_last_error())
        assert release_c(**kw) == code and words in lib.mcamd_last_error(), (kw, lib.mcamd_last_error())
    assert reserve_c(total=-1) == _ext.EINVAL
    assert reserve_c(total=0x7fffffff) == _ext.EUNSUPPORTED
    assert reserve_c(count=None) == _ext.EINVAL and reserve_c(slots=None) == _ext.EINVAL
    assert reserve_c(n_rows=0) == _ext.EINVAL and b"without a row" in lib.mcamd_last_error()
    assert release_c(m=-1) == _ext.EINVAL
    assert release_c(m=0) == _ext.OK and release_c(n_rows=0) == _ext.OK


def test_step_refuses():
    lib = _ext.lib()

    def step(k=FAKE, v=FAKE, D=128, page=16, stride=None, n_pages=4, total=3, q_tok=1024, k_tok=256, eps=1e-6,
             scale=1.2, dtype=_ext.BF16, slots=FAKE, positions=FAKE):
        return lib.mcamd_qk_rope_norm_append_paged(
            FAKE, q_tok, k, k_tok, v, k_tok, FAKE, FAKE, 64, positions, slots, FAKE, FAKE, FAKE, total, 8, 2, D,
            n_pages, page, page * 2 * D if stride is None else stride, eps, scale, dtype, None)

    for kw, code, words in ((dict(D=127), _ext.EUNSUPPORTED, b"even"), (dict(D=258), _ext.EUNSUPPORTED, b"256"),
                            (dict(k=None), _ext.EINVAL, b"both k and v"), (dict(dtype=5), _ext.EINVAL, b"dtype"),
                            (dict(page=20), _ext.EINVAL, b"power of two"),
                            (dict(stride=100), _ext.EINVAL, b"page_stride"),
                            (dict(n_pages=0), _ext.EINVAL, b"empty"), (dict(total=-1), _ext.EINVAL, b"positive"),
                            (dict(q_tok=1000), _ext.EINVAL, b"token stride"),
                            (dict(k_tok=255), _ext.EINVAL, b"token stride"),
                            (dict(eps=-1.0), _ext.EINVAL, b"eps"), (dict(scale=float("inf")), _ext.EINVAL, b"scale"),
                            (dict(total=1 << 31), _ext.EUNSUPPORTED, b"too large"),
                            (dict(slots=None), _ext.EINVAL, b"null"), (dict(positions=None), _ext.EINVAL, b"null")):
        assert step(**kw) == code and words in lib.mcamd_last_error(), (kw, lib.mcamd_last_error())
    assert step(total=0) == _ext.OK


def test_cpu_tensors_are_refused():
    z = torch.zeros(2, dtype=torch.int32)
    pages = torch.zeros(4, 16, 1, 64)
    with pytest.raises(RuntimeError, match="ROCm device"):
        paged_reserve(torch.zeros(2, 3, dtype=torch.int32), z, z, z, z[:1], total=1, page_size=16)
    with pytest.raises(RuntimeError, match="ROCm device"):
        paged_release(torch.zeros(2, 3, dtype=torch.int32), z, z, z, z[:1], page_size=16)
    with pytest.raises(RuntimeError, match="ROCm device"):
        flash_attn.flash_attn_paged_with_kvcache(torch.zeros(2, 1, 1, 64), pages, pages,
                                                 block_table=torch.zeros(2, 3, dtype=torch.int32),
                                                 cache_seqlens=z)
    with pytest.raises(RuntimeError, match="ROCm device"):
        rope_norm_scale_append_paged(torch.zeros(2, 1, 64), torch.zeros(4, 32), torch.zeros(4, 32), z)


def test_page_sizes_and_pools():
    for n in (16, 32, 1024):
        assert check_page_size(n) == n
    for n in (0, 8, 15, 24, 48, -16):
        with pytest.raises(ValueError, match="power of two"):
            check_page_size(n)
    dev = torch.device("cpu")
    pages = torch.zeros(3, 5, 16, 2, 64)
    assert check_pages(pages[1], pages[2], 2, 64, torch.float32, dev) == (5, 16, 16 * 2 * 64)
    assert check_pages(pages[:, 0], pages[:, 1], None, 64, torch.float32, dev) == (3, 16, 5 * 16 * 2 * 64)
    for k, v, Hk, D in ((pages[0], pages[0, :4], 2, 64), (pages[0], pages[0], 1, 64), (pages[0], pages[0], 2, 32),
                        (pages, pages, 2, 64), (pages[0, :0], pages[0, :0], 2, 64),
                        (pages[0].transpose(1, 2), pages[0].transpose(1, 2), 16, 64),
                        (pages[0], pages[:, 0][:, None].expand(3, 5, 16, 2, 64)[0], 2, 64)):
        with pytest.raises(ValueError):
            check_pages(k, v, Hk, D, torch.float32, dev)
    with pytest.raises(TypeError):
        check_pages(pages[0], pages[0], 2, 64, torch.bfloat16, dev)


def test_the_plan_oracle_keeps_every_page():
    """Rows that end and start anew: each page is free or in one line, a refused row changes nothing."""
    g = torch.Generator().manual_seed(0)
    table, lens, free, count = [[-1] * 5 for _ in range(6)], [0] * 6, list(range(20)), [20]
    for _ in range(50):
        done = torch.randperm(6, generator=g)[:2].tolist()
        release(table, lens, done, free, count, 16)
        new = torch.randint(0, 50, (6,), generator=g).tolist()
        slots, positions, cu, refused = reserve(table, lens, new, free, count, sum(new), 16)
        assert cu[-1] == len(slots) == len(positions) == sum(new)
        for b, t in enumerate(new):
            if t and slots[cu[b]] >= 0:
                assert positions[cu[b]] == lens[b]
                lens[b] += t
        held = [p for line in table for p in line if p >= 0]
        assert sorted(held + free[:count[0]]) == list(range(20))
        assert len(set(s for s in slots if s >= 0)) == sum(s >= 0 for s in slots)
