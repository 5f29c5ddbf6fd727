"""What the 8-bit operators refuse on the host and how their sources are laid out, without a GPU."""

import re
from pathlib import Path


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
