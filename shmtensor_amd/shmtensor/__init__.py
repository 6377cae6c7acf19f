"""Mirror of the reference's `shmtensor` Python package
(python/shmtensor/__init__.py:1-4): host tensor providers and the GPU
sampling dataloader on top of the `ShmTensorLib` operators. PagedCache (a key/value
cache in pages, 4 bits a value) has no counterpart there."""
from .. import install_aliases as _install_aliases

capi = _install_aliases()

from .disk_tensor import DiskTensor  # noqa: E402
from .paged_cache import PagedCache  # noqa: E402
from .shm_tensor import ShmTensor  # noqa: E402
from .sampling import GPUSamplingDataloader  # noqa: E402

__all__ = ["DiskTensor", "ShmTensor", "GPUSamplingDataloader", "PagedCache", "capi"]
