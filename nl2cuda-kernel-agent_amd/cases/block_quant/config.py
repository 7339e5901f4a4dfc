"""Sizes and parameters of the block quantisation case: M rows of K numbers
(environment: BQ_M, BQ_K)."""

import os

import torch

SIZES = (int(os.environ.get("BQ_M", "1024")), int(os.environ.get("BQ_K", "2048")))
PARAMS = {"scale_dtype": torch.float8_e8m0fnu}
GRAD_INPUTS = ()
DTYPE = "float32"
