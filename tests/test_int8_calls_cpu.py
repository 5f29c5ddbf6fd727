"""What the 8-bit operators refuse on the host and how their sources are laid out, without a GPU."""

import re
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad

from rdna3_fastmm import int8

BF16 = torch.bfloat16
SOURCES = Path(__file__).resolve().parent.parent / "rdna3-fastmm_b200" / "csrc"


def _kernels(source):
    """Name and body of each kernel of a source file."""
    for part in source.split("__global__")[1:]:
        name = re.search(r"(\w+)\s*\(\s*const", part[part.index("void"):].replace("__launch_bounds__", "", 1)).group(1)
        yield name, part


def test_the_next_kernel_starts_after_tensor_memory_is_allocated():
    """A CTA set up early allocates its own columns before it waits."""
    found = []
    for path in sorted(SOURCES.glob("*.cuh")):
        for name, body in _kernels(path.read_text()):
            if "let_next_kernel_start();" not in body or "tmem_alloc" not in body:
                continue
            found.append(name)
            allocated = body.index("tmem_alloc")
            barrier = min(at for at in (body.find(b, allocated) for b in ("__syncthreads();", "cluster_sync_all();")) if at > 0)
            assert body.index("let_next_kernel_start();") > barrier, name
    assert found == ["int8_linear_kernel", "int8_linear_pair_kernel"]


def _plan(rows, inner, columns, dtype=BF16):
    """A plan over CPU tensors, for its checks alone."""
    plan = int8.Int8Plan.__new__(int8.Int8Plan)
    plan.rows, plan.inner, plan.columns = rows, inner, columns
    plan.device, plan.dtype = torch.device("cpu"), dtype
    return plan


def _operands(rows, inner, columns):
    workspace = int8.Int8Workspace("int8-v1", BF16, torch.zeros((rows, inner), dtype=torch.int8), torch.zeros(rows))
    packed = int8.Int8PackedWeight("int8-v1", BF16, torch.zeros((columns, inner), dtype=torch.int8),
                                   torch.zeros(columns), (columns, inner))
    return workspace, packed


@pytest.mark.parametrize("with_output", [False, True])
def test_a_bias_in_the_workspace_is_refused(with_output, monkeypatch):
    monkeypatch.setattr(int8, "_output_rows", lambda tensor, *args: int8._input_rows(tensor)[1])  # a CPU output
    plan = _plan(8, 64, 16)
    workspace, packed = _operands(8, 64, 16)
    output = torch.zeros((8, 16), dtype=BF16) if with_output else None
    for bias in (workspace.codes.view(-1)[32:64].view(BF16), workspace.scales.view(BF16),
                 workspace.codes.view(-1).view(BF16)[:64:4], workspace.scales.view(BF16)[5:6].expand(16)):
        with pytest.raises(ValueError, match="overlap"):
            plan._validate_product(workspace, packed, bias, output)
    for bias in (torch.zeros(16, dtype=BF16), torch.zeros((16, 3), dtype=BF16)[:, 1]):
        plan._validate_product(workspace, packed, bias, output)


def test_rows_of_tensors_that_are_not_dense():
    def touched(tensor):
        ptr, rows, inner, pitch, size = int8._touched_rows(tensor)
        return (ptr - buffer.data_ptr()) // size, rows, inner, pitch

    buffer = torch.zeros((6, 20))
    assert touched(buffer[1:4, 2:5]) == (22, 3, 3, 20)
    assert touched(buffer[1:4, 2:9:3]) == (22, 3, 7, 20)
    assert touched(buffer[1:4, 2:5].t()) == (22, 3, 3, 20)
    assert touched(buffer[1, 2:3].expand(4, 5)) == (22, 1, 1, 1)
    assert touched(buffer[1:2].expand(4, 20)) == (20, 20, 1, 1)
    assert touched(buffer.view(-1)[7::11]) == (7, 11, 1, 11)
    assert touched(buffer.as_strided((3, 8), (5, 1))) == (0, 1, 18, 18)
    assert touched(buffer[:, ::2][:0])[1] == 0
    # beside each other in the rows of one buffer
    assert not int8._rows_overlap(int8._touched_rows(buffer[:, :10:2]), int8._touched_rows(buffer[:, 10:]))
    assert int8._rows_overlap(int8._touched_rows(buffer[:, :12:2]), int8._touched_rows(buffer[:, 10:]))


@torch.enable_grad()  # whatever the mode that a test before left behind
def test_gradients_tangents_and_negated_views_are_refused():
    x, codes = torch.zeros(3, 4), torch.zeros((3, 4), dtype=torch.int8)
    int8._refuse_unread(x, None, codes)
    leaf = x.clone().requires_grad_(True)
    for refused in (leaf, leaf * 2, torch._neg_view(x), torch._neg_view(codes)):
        with pytest.raises(ValueError):
            int8._refuse_unread(x, None, refused)
    with torch.no_grad():
        int8._refuse_unread(leaf, leaf * 2)
    with forward_ad.dual_level():
        int8._refuse_unread(x, codes)
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for operand in (dual, dual * 2, dual.t()):
            with pytest.raises(ValueError, match="autograd"):
                int8._refuse_unread(x, operand)
            with torch.no_grad(), pytest.raises(ValueError, match="autograd"):  # which leaves tangents alone
                int8._refuse_unread(x, operand)
    int8._refuse_unread(x)


def test_torch_operators_refuse_forward_transforms():
    def call(x):
        int8._refuse_transforms()
        return x

    x = torch.zeros(3)
    torch.func.vmap(call)(x)
    torch.func.grad(lambda x: call(x).sum())(x)
    for transform in (lambda: torch.func.jvp(call, (x,), (x,)), lambda: torch.func.jacfwd(call)(x)):
        with pytest.raises(ValueError, match="jvp"):
            transform()
    call(x)
