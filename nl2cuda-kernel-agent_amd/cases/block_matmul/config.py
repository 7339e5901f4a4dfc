"""Sizes and parameters of the block-scaled product: M rows times a weight of N
rows, K numbers each (environment: BM_M, BM_N, BM_K)."""

import os

import torch

SIZES = (int(os.environ.get("BM_M", "512")), int(os.environ.get("BM_N", "1024")),
         int(os.environ.get("BM_K", "2048")))
PARAMS = {"scale_dtype": torch.float8_e8m0fnu}
GRAD_INPUTS = ("X", "W")
DTYPE = "float32"
