"""ctypes declarations of every symbol of include/mgrid_norm.h: the C ABI without its torch binding."""
import ctypes as C

from multigrid_amd import fused_ops

P, L, I = C.c_void_p, C.c_int64, C.c_int
# name -> (restype, argtypes)
SYMBOLS = {
    'mgnn_layer_norm': (I, [P, L, P, P, P, P, L, L, I, C.c_double, I, I, P]),
    'mgnn_layer_norm_workspace': (L, [L, L, I, I]),
    'mgnn_layer_norm_backward': (I, [P, L, P, P, P, P, P, P, P, L, L, L, I, I, I, P]),
    'mgnn_grad_norm_workspace': (L, [P, P, L, L]),
    'mgnn_grad_norm': (I, [P, P, P, L, L, P, P, L, P]),
    'mgnn_clip_grads': (I, [P, P, P, P, L, L, C.c_double, P, P, L, P]),
}


def load():
  lib = C.CDLL(fused_ops.LIB_PATH)
  for name, (res, args) in SYMBOLS.items():
    fn = getattr(lib, name)
    fn.restype, fn.argtypes = res, args
  return lib
