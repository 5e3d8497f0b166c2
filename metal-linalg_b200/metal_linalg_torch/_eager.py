"""Which calls may hand their tensors' addresses to the library at once.

The operators of _delta.py and _fp8.py are torch custom operators, and eager calls on plain tensors go round the dispatcher
(about 10 us a call). Whatever watches or replaces operators has to see them, so that every other call takes the dispatcher:
torch.compile and export, `make_fx` and fake tensors (dispatch modes, pre-dispatch tracing), `torch.jit.trace`, the transforms of
`torch.func`, tensor subclasses and meta tensors.
"""
import torch
import torch.autograd.forward_ad as _forward_ad
from torch import Tensor

_PLAIN = frozenset((Tensor, torch.nn.Parameter, type(None)))
_is_compiling = torch.compiler.is_compiling
_dispatch_modes = torch._C._len_torch_dispatch_stack
_is_tracing = torch._C._is_tracing
_transforms = torch._C._functorch.peek_interpreter_stack
_is_included = torch._C._dispatch_tls_is_dispatch_key_included
_PRE_DISPATCH = torch._C.DispatchKey.PreDispatch


def direct(name, *tensors):
    """Whether operator `name` may use the addresses of `tensors` (None allowed behind the first). Refuses forward-mode
    tangents, which no operator here carries on."""
    if _is_compiling():
        return False
    if _forward_ad._current_level >= 0 and any(x is not None and _forward_ad.unpack_dual(x).tangent is not None for x in tensors):
        raise RuntimeError(f"metal_linalg_torch.{name}: forward-mode derivatives are not supported")
    return (not _dispatch_modes() and not _is_tracing() and _transforms() is None and not _is_included(_PRE_DISPATCH)
            and _PLAIN.issuperset(map(type, tensors)) and not tensors[0].is_meta)
