"""pytest plugin: the token operators' GPU tests on the CPU build of their kernels
($CPU_KERNELS, see tests/test_token_ops_cpu.py)."""
import ctypes
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path[:0] = [ROOT, os.path.join(ROOT, "multimodal-ghm_amd"), os.path.join(ROOT, "tests")]

import torch  # noqa: E402

from ghmclip import _native  # noqa: E402
from ghmclip.models import token_ops  # noqa: E402

torch.set_num_threads(1)
_lib = ctypes.CDLL(os.environ["CPU_KERNELS"])
for _name, _args in _native.HIP_SIGNATURES.items():
    if _name.startswith(("ghm_token_logprobs", "ghm_distill", "ghm_embed_rows")):
        getattr(_lib, _name).argtypes = _args
        getattr(_lib, _name).restype = _native._RESTYPE.get(_name, ctypes.c_int)
_lib.ghm_last_error_string.restype = ctypes.c_char_p
_native._hip = _lib
token_ops.require_hip = lambda t: None
token_ops._call = lambda device, name, *args: _native.call(name, *args, None)
torch.cuda.is_available = lambda: True
torch.cuda.synchronize = torch.cuda.empty_cache = lambda *a: None


def pytest_collection_modifyitems(items):
    for item in items:
        item.module.DEV = "cpu"
