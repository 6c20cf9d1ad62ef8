"""linrec_amd: first-order linear recurrence y[l] = y[l-1]*c[l] + x[l] for MI355X (gfx950).

    import linrec_amd
    y = linrec_amd.linrec(inputs, coeffs, reverse=False)

and the operators of a recurrent layer around it (layers.py): gated_linrec, gated_linrec_step, group_norm_act, embedding.

Drop-in for `linrec.linrec` of safelix/linrec (linrec/__init__.py:3-11).  Importing this package
loads the HIP library; if it has not been built the import fails (there is no Triton or eager
stand-in for device tensors).
"""
from . import _native

_native.lib()  # fail at import, not at first call, when the library is missing

from .ops import linrec, linrec_bwd, linrec_fwd, linrec_pipe, linrec_ref, linrec_tile  # noqa: E402
from .layers import embedding, gated_linrec, gated_linrec_step, group_norm_act  # noqa: E402
from ._native import Tuning, kernel_attrs, kernel_table, plan  # noqa: E402

__all__ = ["linrec", "linrec_fwd", "linrec_bwd", "linrec_pipe", "linrec_tile", "linrec_ref",
           "gated_linrec", "gated_linrec_step", "group_norm_act", "embedding",
           "Tuning", "plan", "kernel_table", "kernel_attrs"]
