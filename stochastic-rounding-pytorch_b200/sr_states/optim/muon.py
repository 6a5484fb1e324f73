"""Muon: momentum whose update is orthogonalised, with a configurable momentum format.

No counterpart in the reference; constructor options, per-group formats,
counter-hash rounding and checkpoints follow the other optimizers of the package.
"""

from __future__ import annotations

from ._state import StateOptimizer


class MuonSR(StateOptimizer):
    """u' = u*momentum + g; v = u'*momentum + g (``nesterov``) or u';
    p' = p*(1 - lr*weight_decay) - lr*s*O, O the Newton-Schulz orthogonalisation
    of v.  u' is stored with its format (BF16 stochastic by default).

    For matrices: parameters of two or more dimensions, those after the first
    flattened; embeddings, norms and biases belong to AdamW.  ``scale`` names the
    shape's factor s: ``"spectral"`` sqrt(max(1, rows / columns)) or ``"rms"``
    0.2 * sqrt(max(rows, columns)).  Parameters must be CUDA tensors on sm_100a.
    """

    _state_names = ("momentum_buffer",)
    _uses_step = False
    _rounding_backend = "cuda"

    def __init__(self, params, lr=0.02, momentum=0.95, weight_decay=0.0, *, nesterov=True,
                 scale="spectral", ns_steps=5, ns_coefficients=(3.4445, -4.7750, 2.0315),
                 eps=1e-7, state_format=None, state_dtype=None, rounding=None, seed=0):
        super().__init__(params, {"lr": lr, "momentum": momentum, "weight_decay": weight_decay,
                                  "nesterov": bool(nesterov), "scale": scale,
                                  "ns_steps": ns_steps,
                                  "ns_coefficients": tuple(ns_coefficients), "eps": eps},
                         state_format=state_format, state_dtype=state_dtype, rounding=rounding,
                         seed=seed)

    def _validate_group(self, group):
        from ..cuda.muon import check_matrix, check_muon, newton_settings  # imports this module

        check_muon(group["lr"], group["momentum"], group["weight_decay"], group["scale"])
        newton_settings(group["ns_steps"], group["ns_coefficients"], group["eps"])
        parameters = group.get("params", ())
        if isinstance(parameters, (list, tuple)):
            for parameter in parameters:
                if hasattr(parameter, "dim"):  # a checkpoint's group holds indices
                    check_matrix(parameter)

    def state_dict(self):
        """The optimizer's state; RuntimeError if a product kernel of a step gave up (waits
        for the parameters' devices)."""
        from ..cuda.muon import check_products

        for device in {p.device for p in self.state if p.device.type == "cuda"}:
            check_products(device)
        return super().state_dict()

    def _step_group(self, group, formats, items, rng_step):
        from ..cuda.muon import muon_group_step  # the backend imports this module

        muon_group_step(self, group, formats, items, rng_step)


class MuonRN(MuonSR):
    """Muon storing the momentum with round-to-nearest-even."""

    _forced_rounding = "nearest"
