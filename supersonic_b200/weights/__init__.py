"""Weight sources: safetensors by tensor name, seeded random weights, model folders; matrices in 4 bits."""
from .fp4 import Fp4Matrix
from .safetensors_io import SafetensorsError, SafetensorsFile, write_safetensors
from .store import (RandomWeightStore, WeightError, WeightStore, random_store, random_tensors,
                    write_model_folder)

__all__ = ["Fp4Matrix", "SafetensorsError", "SafetensorsFile", "write_safetensors", "WeightError",
           "WeightStore", "RandomWeightStore", "random_store", "random_tensors", "write_model_folder"]
