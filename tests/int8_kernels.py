"""Which 8-bit kernels a call launches, for tests that are about one of them."""

import re

import torch


def kernels_of(call):
    """The names of the ``int8_*`` kernels that ``call`` launches, without template arguments."""
    call()  # what a first call sets up
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as profile:
        call()
        torch.cuda.synchronize()
    names = (re.search(r"int8_\w+_kernel", event.name) for event in profile.events())
    return [name.group() for name in names if name]
