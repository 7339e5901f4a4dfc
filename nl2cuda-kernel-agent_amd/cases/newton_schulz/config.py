"""Sizes and parameters of the Newton-Schulz case: `count` matrices m x n
(environment: NS_COUNT, NS_M, NS_N)."""

import os

SIZES = (int(os.environ.get("NS_COUNT", "2")), int(os.environ.get("NS_M", "512")),
         int(os.environ.get("NS_N", "1024")))
PARAMS = {"steps": 5, "coefficients": (3.4445, -4.7750, 2.0315), "eps": 1e-7}
GRAD_INPUTS = ()
DTYPE = "float32"
