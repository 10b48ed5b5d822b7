"""Adapter training: an autograd forward over the frozen model, in plain PyTorch or
(``TrainParameters.fused``) on the training operators."""
from .forward import MaskStream, TrainableLoRA, train_forward, train_hidden  # noqa: F401
from .lora_train import (Progress, TrainParameters, evaluate, iterate_batches, load_lora_data,  # noqa: F401
                         load_lora_file, loss_fn, train)
