"""The words that pages are copied in: no wider claim of alignment than the layers' bases bear."""

import re
import subprocess

import pytest
import torch

from everserve_amd import build
from everserve_amd.state.fp4 import Fp4Cache, cache_shape
from everserve_amd.state.pages import PageMover
from tests.cases import LAYOUTS, bits

# bytes that a layer's first element lies off the allocation's start (16 bytes and more)
OFFSETS = [(64, 4), (128, 4), (128, 8), (128, 12), (136, 4)]


def fp4_layers(layout, d, off, device, n_layers=2):
    """4-bit caches whose bases lie ``off`` bytes past a multiple of 16, of random bytes."""
    g = torch.Generator().manual_seed(d + off)
    shape = cache_shape(layout, 6, 16, 2, d)
    n = torch.Size(shape).numel()
    flat = torch.randint(0, 256, (n_layers, (n + off + 15) // 16 * 16), dtype=torch.uint8,
                         generator=g).to(device)
    return [row[off:off + n].view(shape) for row in flat]


def test_the_copys_words_claim_no_alignment():
    """A word is chosen from a page's strides and runs, and the bases are known to the device alone:
    every load and store of a word must be one that may start at any byte."""
    src = build.CSRC / "pages.hip"
    ir = subprocess.run(
        [build.hipcc(), *build.HIPCC_FLAGS, "--offload-arch=gfx950", "--offload-device-only", "-S",
         "-emit-llvm", f"-I{build.INCLUDE}", f"-I{build.CSRC}", str(src), "-o", "-"],
        check=True, stdout=subprocess.PIPE, stderr=subprocess.DEVNULL, text=True).stdout
    moves = [line for line in ir.splitlines() if "!nontemporal" in line]
    assert len(moves) >= 10  # a load and a store of each of five word sizes
    assert {re.search(r"align (\d+)", line).group(1) for line in moves} == {"1"}


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("d,off", OFFSETS)
def test_four_bit_caches_on_any_dword_are_taken(layout, d, off):
    layers = fp4_layers(layout, d, off, "cpu")
    assert all(t.data_ptr() % 16 == off % 16 for t in layers)
    mover = PageMover(layers, layout)
    assert mover.num_blocks == Fp4Cache(layers[0], d, layout).num_blocks == 6


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("d,off", OFFSETS)
def test_pages_of_four_bit_caches_on_any_dword_are_copied(ext, layout, d, off):
    gpu = fp4_layers(layout, d, off, "cuda")
    copy_and_check(gpu, layout)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype,off", [(torch.uint8, 1), (torch.uint8, 7), (torch.bfloat16, 1),
                                       (torch.bfloat16, 3), (torch.float32, 1)])
def test_pages_on_any_element_are_copied(ext, layout, dtype, off):
    # a head's rows of 18 elements: no stride is whole words of 16 bytes, whole pages are
    shape = {"kv_first": (2, 6, 8, 2, 18), "blocks_first": (6, 2, 8, 2, 18),
             "combined": (6, 2, 8, 36)}[layout]
    n = torch.Size(shape).numel()
    g = torch.Generator().manual_seed(off)
    flat = (100 * torch.rand(2, n + 16, generator=g)).to(dtype).cuda()
    gpu = [row[off:off + n].view(shape) for row in flat]
    around = flat.clone()
    copy_and_check(gpu, layout)
    for row, old in zip(flat, around):  # nothing else was written
        assert torch.equal(row[:off], old[:off]) and torch.equal(row[off + n:], old[off + n:])


def copy_and_check(gpu, layout):
    want = [t.cpu().clone() for t in gpu]
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 5, 2], [3, 1, 4])]
    PageMover(gpu, layout).copy(*ints)
    for t in want:
        p = t.transpose(0, 1) if layout == "kv_first" else t
        for s, d in ((0, 3), (5, 1), (2, 4)):
            p[d] = p[s].clone()
    torch.cuda.synchronize()
    for a, b in zip(gpu, want):
        assert (bits(a) == bits(b)).all()
