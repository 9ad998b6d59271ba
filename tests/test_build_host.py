"""CPU: what makes the libraries be rebuilt, and what a build refuses."""
import pytest
import torch

import q3attn.build as build


def test_another_torch_means_another_build(monkeypatch):
    """The bindings are compiled against torch's C++ interface: a library built for another torch is not up to date."""
    here = build.source_digest()
    assert build.source_digest() == here
    monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    assert build.source_digest() != here and not build.up_to_date()
    monkeypatch.undo()
    monkeypatch.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI)
    assert build.source_digest() != here


def log(*kernels):
    return "\n".join(f"ptxas info    : Compiling entry function '_ZN2q317paged_tree_kernelILb{f}ELb{d}ELi{s}ELi{n}ELi3EEEvT' for 'sm_100a'\n"
                     f"ptxas info    : Function properties for x\n    0 bytes stack frame, 0 bytes spill stores\n"
                     f"ptxas info    : Used {r} registers, used 1 barriers" for f, d, s, n, r in kernels)


def test_the_build_says_when_a_register_split_does_not_fit():
    good = [(1, 0, 2, 1, 96), (1, 1, 1, 2, 168), (0, 1, 1, 1, 121)]     # one stream, four tokens: nothing is moved
    build.check_registers(log(*good))
    for bad in ((1, 1, 2, 1, 94), (0, 1, 1, 2, 160)):
        with pytest.raises(RuntimeError, match="register split"):
            build.check_registers(log(good[0], bad, good[2]))
    with pytest.raises(RuntimeError, match="names no kernel"):
        build.check_registers("")
