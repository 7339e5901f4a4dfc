"""Sizes and parameters of the policy loss case: B answers of S tokens over V
classes (environment: POLICY_B, POLICY_S, POLICY_V)."""

import os

SIZES = (int(os.environ.get("POLICY_B", "4")), int(os.environ.get("POLICY_S", "256")),
         int(os.environ.get("POLICY_V", "8192")))
PARAMS = {"clip_low": 0.2, "clip_high": 0.28, "kl_coef": 0.04, "temperature": 1.0}
GRAD_INPUTS = ("logits",)
DTYPE = "float32"
