"""What the operators that cast their arguments under autocast have in common."""
from __future__ import annotations

from typing import Optional

import torch

from . import _ext


def check_cast_leaves(*tensors: Optional[torch.Tensor]) -> None:
    """Refuse a captured call whose leaves a living eager graph keeps, before a
    cast hides them: their gradients would go to them on that graph's stream,
    out of the capture."""
    if torch.cuda.is_current_stream_capturing():
        _ext().check_cast_leaves([t for t in tensors if t is not None])
