"""ctypes mirrors of the argument structs of layer norm and the 8-bit products (include/spb_hip.h)."""
import ctypes as C

vp, i32, i64, f32 = C.c_void_p, C.c_int, C.c_longlong, C.c_float


class LayerNormArgs(C.Structure):
    _fields_ = [("X", vp), ("G", vp), ("gamma", vp), ("beta", vp), ("Y", vp), ("mean", vp), ("rstd", vp), ("dgamma", vp), ("dbeta", vp),
                ("part", vp), ("part_cap", i64), ("M", i64), ("ldx", i64), ("ldg", i64), ("ldy", i64), ("C", i32), ("eps", f32),
                ("accumulate", i32)]


class Gemm8Args(C.Structure):
    _fields_ = [("A", vp), ("As", vp), ("B", vp), ("Bs", vp), ("bias", vp), ("Y", vp), ("ws", vp), ("ws_bytes", i64), ("M", i64), ("ldy", i64),
                ("N", i32), ("K", i32), ("b_block_rows", i32)]


class Wgrad8Args(C.Structure):
    _fields_ = [("G", vp), ("X", vp), ("Xs", vp), ("dW", vp), ("ws", vp), ("ws_bytes", i64), ("M", i64), ("ldg", i64), ("ldw", i64),
                ("N", i32), ("K", i32), ("accumulate", i32)]
