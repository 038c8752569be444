"""Neural-network modules and optimizers."""

from .module import (
    Attention,
    Dropout,
    Embedding,
    KeyValueCache,
    Linear,
    Module,
    ReLU,
    RMSNorm,
    Sequential,
    Sigmoid,
    Tanh,
)
from .optimizers import AdamW, GradientDescent, Optimizer

__all__ = ["AdamW", "Attention", "Dropout", "Embedding", "GradientDescent", "KeyValueCache",
           "Linear", "Module", "Optimizer", "RMSNorm", "ReLU", "Sequential", "Sigmoid", "Tanh"]
