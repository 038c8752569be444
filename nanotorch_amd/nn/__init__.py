"""Neural-network modules and optimizers."""

from .module import Dropout, Embedding, Linear, Module, ReLU, Sequential, Sigmoid, Tanh
from .optimizers import GradientDescent, Optimizer

__all__ = ["Dropout", "Embedding", "GradientDescent", "Linear", "Module", "Optimizer", "ReLU",
           "Sequential", "Sigmoid", "Tanh"]
