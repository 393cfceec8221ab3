"""Forward-mode automatic differentiation, which this package has not."""

import torch.autograd.forward_ad as _forward_ad


def refuse_tangents(name, *tensors):
    """Raises ``NotImplementedError`` where one of ``tensors`` (or None)
    carries a tangent: the kernels would return a constant in its place."""
    if _forward_ad._current_level < 0:  # outside every dual level
        return
    for t in tensors:
        if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has no forward-mode derivative")
