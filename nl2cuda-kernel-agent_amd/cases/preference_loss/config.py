"""Sizes and parameters of the preference loss case: N pairs of answers of at
most S tokens over V classes (environment: PREF_N, PREF_S, PREF_V)."""

import os

SIZES = (int(os.environ.get("PREF_N", "2")), int(os.environ.get("PREF_S", "256")),
         int(os.environ.get("PREF_V", "8192")))
PARAMS = {"beta": 0.1, "label_smoothing": 0.0, "average": False}
GRAD_INPUTS = ("logits",)
DTYPE = "float32"
