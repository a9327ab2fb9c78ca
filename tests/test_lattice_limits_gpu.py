"""Lengths and page numbers that the lattice kernels must refuse on the device: lengths next to 2^31, where rounding up to
blocks or pages in 32 bits would wrap and look like a length that fits, and pages outside the pool."""
import pytest
import torch

from lockstep_b200 import decode as D

pytestmark = pytest.mark.gpu
HUGE = (2 ** 31 - 1, 2 ** 31 - 100, 2 ** 31 - 127, 2 ** 31 - 128, 2 ** 30)


def make(dh, sink=False, B=3, L=700):
    g = torch.Generator("cuda").manual_seed(dh)
    draw = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)       # noqa: E731
    k, v = draw(B, 2, L, dh), draw(B, 2, L, dh)
    return k, v, D.contiguous_kv(k, v, sink=sink), draw(B, 8, dh)


def same(a, b):
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


@pytest.mark.parametrize("length", HUGE)
@pytest.mark.parametrize("dh", [64, 128])
def test_huge_lengths_are_flagged(dh, length):
    k, v, kv, q = make(dh)
    want = D.decode(q, kv)
    kv.block_table[1:, :40] = kv.block_table[0, :40].clone()     # the first 640 tokens are shared
    kv.ek[1:, :, :5], kv.ev[1:, :, :5] = kv.ek[0, :, :5].clone(), kv.ev[0, :, :5].clone()
    shared = D.decode(q, kv)
    assert same(D.decode_shared(q, kv, 640), shared) and same(shared[0], want[0])
    kv.seq_lens[1] = length
    for n in (0, 640):
        out = torch.full_like(q, 3.0)
        with pytest.raises(RuntimeError, match="bits 0x4 "):
            D.decode_shared(q, kv, n, out=out)
        assert same(out[[0, 2]], shared[[0, 2]]) and (out[1] == 3.0).all()
    rows = length % 128 or 128                                   # its last rows, from a block boundary
    qp = torch.randn(700 + rows, 8, dh, device="cuda").to(torch.bfloat16)
    cu = torch.tensor([0, 700, 700 + rows, 700 + rows], dtype=torch.int32, device="cuda")
    act = torch.tensor([True, False, False], device="cuda")
    alone = D.prefill_paged(qp, kv, cu, active=act)
    out = torch.full_like(qp, 3.0)
    with pytest.raises(RuntimeError, match="bits 0x4 "):
        D.prefill_paged(qp, kv, cu, out=out)
    assert same(out[:700], alone[:700]) and (out[700:] == 3.0).all()


@pytest.mark.parametrize("length", HUGE)
@pytest.mark.parametrize("dh", [64, 128])
def test_the_writers_flag_huge_lengths(dh, length):
    k, v, kv, q = make(dh)
    keep = [x.clone() for x in (kv.k8p, kv.v8p, kv.ek, kv.ev)]
    lens = torch.tensor([700, length, 700], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="bits 0x4 "):
        D.build_paged_kv(k, v, lens, kv.block_table, kv.num_pages, out=kv)
    with pytest.raises(RuntimeError, match="bits 0x4 "):
        D.append_kv(kv, k, v, lens)
    with pytest.raises(RuntimeError, match="bits 0x4 "):         # rows off the 16-byte grid: the general writer
        D.build_paged_kv(k.transpose(2, 3).contiguous().transpose(2, 3), v.transpose(2, 3).contiguous().transpose(2, 3), lens,
                         kv.block_table, kv.num_pages, out=kv)
    assert all(torch.equal(a, b) for a, b in zip(keep, (kv.k8p, kv.v8p, kv.ek, kv.ev)))


@pytest.mark.parametrize("page", [-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("dh", [64, 128])
def test_a_first_page_outside_the_pool_with_the_sink(dh, page):
    """Key 0's own term reads its value row again in the refold: page 0 stands in there too."""
    k, v, kv, q = make(dh, sink=True)
    kv.block_table[1, 0] = 0
    want = D.decode(q, kv)
    kv.block_table[1, 0] = page
    for n in (0, 100):
        out = torch.zeros_like(q)
        with pytest.raises(RuntimeError, match="bits 0x4 "):
            D.decode_shared(q, kv, n, out=out)
        assert same(out, want)
    with pytest.raises(RuntimeError, match="bits 0x4 "):
        D.decode(q, kv)
