"""Newton-Schulz case: exposes ``CASE`` at the config module's sizes and
``make_case`` for others."""

import os

from framework.case import Case
from cases.newton_schulz import config
from cases.newton_schulz.reference import make_inputs, make_inputs_for, reference_forward


def _load_description():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "description.md")
    with open(path, encoding="utf-8") as f:
        return f.read()


def make_case(*sizes, **params):
    """A Case at other sizes (those of config.SIZES, in order) and parameters."""
    return Case(
        name="newton_schulz",
        description=_load_description(),
        params={**config.PARAMS, **params},
        grad_inputs=list(config.GRAD_INPUTS),
        dtype=config.DTYPE,
        make_inputs=make_inputs_for(*sizes) if sizes else make_inputs,
        reference_forward=reference_forward,
    )


CASE = make_case()
