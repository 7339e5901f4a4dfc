"""Sizes and parameters of the root-mean-square norm case: B rows of D numbers
(environment: RMS_B, RMS_D)."""

import os

SIZES = (int(os.environ.get("RMS_B", "1024")), int(os.environ.get("RMS_D", "2048")))
PARAMS = {"eps": 1e-6}
GRAD_INPUTS = ("X", "R", "W")
DTYPE = "float32"
