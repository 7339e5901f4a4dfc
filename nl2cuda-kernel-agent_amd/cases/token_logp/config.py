"""Sizes and parameters of the token log-probability case: B sequences of S
tokens over V classes (environment: LOGP_B, LOGP_S, LOGP_V)."""

import os

SIZES = (int(os.environ.get("LOGP_B", "4")), int(os.environ.get("LOGP_S", "256")),
         int(os.environ.get("LOGP_V", "8192")))
PARAMS = {"temperature": 1.0}
GRAD_INPUTS = ("logits",)
DTYPE = "float32"
