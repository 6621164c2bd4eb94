"""Host-side mirror of the reference tensor-math interface on torch CUDA tensors.

Names, argument order and error behaviour follow the reference's static classes
(cuda/ctensorconv.cu.h:63-66, cuda/ctensormath.cu.h:92-135, cuda/ctensorapplyfunc.cu.h:78-90):
the output tensor comes first and is pre-sized by the caller, tensors are 4-D (W,Z,Y,X) fp32,
operands broadcast over W by modulo, and a shape error raises B200Error carrying the library's
message (the reference throws a C string).  All work happens in libb200conv.so on the current
torch CUDA stream; nothing here computes.
"""
import ctypes as C

import torch

from .lib import ConvGeom, load

TF32X3, TF32, FP32 = 0, 1, 2
PATH_SIMT, PATH_TCGEN05 = 1, 2
ACT = {"sigmoid": 0, "relu": 1, "leaky_relu": 2, "linear": 3, "tanh": 4, "gelu": 5}


class B200Error(RuntimeError):
    def __init__(self, code, text):
        super().__init__(f"b200conv error {code}: {text}")
        self.code = code


def _check(code):
    if code != 0:
        raise B200Error(code, load().b200_last_error().decode(errors="replace"))


def _t(x, name="tensor"):
    if not (isinstance(x, torch.Tensor) and x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()):
        raise B200Error(2, f"{name} must be a contiguous fp32 CUDA tensor")
    return x


def _ptr(x):
    return C.c_void_p(x.data_ptr()) if x is not None else None


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def set_precision(mode):
    _check(load().b200_set_precision(mode))


def get_precision():
    return load().b200_get_precision()


def last_path():
    return load().b200_last_path()


def stream_status():
    """Synchronises the current stream and raises if a kernel recorded a failure."""
    _check(load().b200_stream_status(_stream()))


def geom(in_z, in_y, in_x, kernel_amount, kernel_x, kernel_y, stride_x, stride_y, padding_x, padding_y, out_y=None, out_x=None):
    if out_y is None:
        out_y = (in_y - kernel_y + 2 * padding_y) // stride_y + 1
    if out_x is None:
        out_x = (in_x - kernel_x + 2 * padding_x) // stride_x + 1
    return ConvGeom(in_z, in_y, in_x, kernel_amount, kernel_y, kernel_x, stride_y, stride_x, padding_y, padding_x, out_y, out_x)


# ---- layer normalisation and 8-bit checkpoints: activations in fp32, bf16 or fp16, as matrices of rows --------------------------

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_F32 = torch.float32
_MOST_ROWS = (1 << 31) - 65536       # rows, and values in a row (b200conv.h)


# The calls below take a few microseconds, most of them spent here: each looks the device up once and hands it on.

def _rows(x, name, dev):
    """(type code, rows, values in a row, pitch) of an activation tensor: its first dimension is the rows, the others (dense)
    are a row.  A 2-D tensor may have any pitch between its rows."""
    kind = _TYPES.get(x.dtype) if isinstance(x, torch.Tensor) else None
    if kind is None or not x.is_cuda:
        raise B200Error(2, f"{name} must be an fp32, bf16 or fp16 CUDA tensor")
    if x.get_device() != dev:
        raise B200Error(2, f"{name} is on {x.device}, the current device is cuda:{dev}")
    shape = x.shape
    if shape and shape[0] > _MOST_ROWS:
        raise B200Error(1, f"{name} has {shape[0]} rows, {_MOST_ROWS} at most")      # (a C int would keep the lower 32 bits)
    if len(shape) == 2 and shape[1]:
        rows, n = shape
        if n > _MOST_ROWS:
            raise B200Error(1, f"{name} has rows of {n} values, {_MOST_ROWS} at most")
        pitch, inner = x.stride()
        if (inner == 1 or n == 1) and (pitch >= n or rows <= 1):
            return kind, rows, n, pitch if pitch > n else n
    if not shape or not x.is_contiguous():
        raise B200Error(2, f"{name} must be contiguous, or a matrix of contiguous rows")
    n = torch.Size(shape[1:]).numel()
    if n > _MOST_ROWS:
        raise B200Error(1, f"{name} has rows of {n} values, {_MOST_ROWS} at most")
    return kind, shape[0], n, n


def _param(x, n, name, dev):
    """The address of x, a contiguous fp32 tensor of n elements on the current device."""
    try:
        if x.dtype is _F32 and x.numel() == n and x.get_device() == dev and x.is_contiguous():
            return x.data_ptr()
    except AttributeError:
        pass
    _t(x, name)
    if x.numel() != n:
        raise B200Error(1, f"{name} must have {n} elements")
    raise B200Error(2, f"{name} is on {x.device}, the current device is cuda:{dev}")


def _like(x, name, want, other, dev):
    """The pitch of x, which must have the type, rows and row length of `other`."""
    got = _rows(x, name, dev)
    if got[0] != want[0]:
        raise B200Error(2, f"{name} must have the type of {other}")
    if got[1:3] != want[1:3]:
        raise B200Error(1, f"{name} must have the size of {other}")
    return got[3]


class Checkpoint8:
    """An activation tensor kept in 8 bits a value (see b200_ckpt8_store in include/b200conv.h for the format): `rows` rows of
    `n` values, 33 bytes for 32 of them.  codes is an int8 tensor [rows, 32 * blocks], exponents a uint8 tensor [rows, blocks],
    blocks = ceil(n / 32); both belong to the caller."""
    __slots__ = ("codes", "exponents", "rows", "n")

    def __init__(self, codes, exponents, n):
        if not (codes.is_cuda and exponents.is_cuda and codes.dtype == torch.int8 and exponents.dtype == torch.uint8 and
                codes.is_contiguous() and exponents.is_contiguous()):
            raise B200Error(2, "codes and exponents must be contiguous int8 and uint8 CUDA tensors")
        if not codes.get_device() == exponents.get_device() == _device():
            raise B200Error(2, "codes and exponents must be on the current device")
        blocks, rows = (n + 31) // 32, codes.shape[0]
        if n < 1 or codes.shape != (rows, 32 * blocks) or exponents.shape != (rows, blocks):
            raise B200Error(1, "codes must be [rows, 32 * blocks] and exponents [rows, blocks], blocks = ceil(n / 32)")
        self.codes, self.exponents, self.rows, self.n = codes, exponents, rows, n

    @classmethod
    def empty(cls, rows, n, device="cuda"):
        blocks = (n + 31) // 32
        return cls(torch.empty(rows, 32 * blocks, dtype=torch.int8, device=device),
                   torch.empty(rows, blocks, dtype=torch.uint8, device=device), n)

    def _here(self, dev):
        """This checkpoint, which must be on the current device."""
        if self.codes.get_device() != dev:
            raise B200Error(2, f"the checkpoint is on {self.codes.device}, the current device is cuda:{dev}")
        return self

    def _match(self, x, name, dev):
        got = _rows(x, name, dev)
        self._here(dev)
        if got[1] != self.rows or got[2] != self.n:
            raise B200Error(1, f"{name} must have {self.rows} rows of {self.n} values")
        return got

    def store(self, x, keep_sign=False):
        """Keeps x.  keep_sign: a negative value never becomes 0 (the derivative of ReLU and LeakyReLU is then exact)."""
        dev = _device()
        kind, rows, n, pitch = self._match(x, "x", dev)
        _check(load().b200_ckpt8_store(self.codes.data_ptr(), self.exponents.data_ptr(), x.data_ptr(), kind, rows, n, pitch,
                                       int(keep_sign), _raw_stream(dev)))
        return self

    def load(self, output):
        """The kept values into `output` (fp32, bf16 or fp16), which is returned."""
        dev = _device()
        kind, rows, n, pitch = self._match(output, "output", dev)
        _check(load().b200_ckpt8_load(output.data_ptr(), self.codes.data_ptr(), self.exponents.data_ptr(), kind, rows, n, pitch,
                                      _raw_stream(dev)))
        return output


class CTensorConv:
    """cuda/ctensorconv.cu.h:63-66."""

    @staticmethod
    def ForwardConvolution(output, image, kernel, kernel_x, kernel_y, kernel_z, kernel_amount, bias,
                           stride_x, stride_y, padding_x, padding_y):
        _t(output), _t(image), _t(kernel), _t(bias)
        if bias.shape[1] != kernel_amount:
            raise B200Error(1, "the number of kernels and biases must match")
        if image.shape[1] != kernel_z:
            raise B200Error(1, "filter depth and image depth must match")
        if kernel.shape[2] != kernel_amount or kernel.shape[3] != kernel_x * kernel_y * kernel_z:
            raise B200Error(1, "kernel tensor must be [Wk,1,K,C*ky*kx]")
        if output.shape[1] != kernel_amount:
            raise B200Error(1, "wrong output depth for convolution")
        g = geom(kernel_z, image.shape[2], image.shape[3], kernel_amount, kernel_x, kernel_y, stride_x, stride_y,
                 padding_x, padding_y, output.shape[2], output.shape[3])
        _check(load().b200_conv_forward(C.byref(g), _ptr(output), output.shape[0], _ptr(image), image.shape[0],
                                        _ptr(kernel), kernel.shape[0], _ptr(bias), bias.shape[0], _stream()))

    @staticmethod
    def BackwardConvolution(output_delta, delta, kernel, kernel_x, kernel_y, kernel_z, kernel_amount, bias,
                            stride_x, stride_y, padding_x, padding_y):
        """bias=None stands for the all-zero bias every reference caller passes."""
        _t(output_delta), _t(delta), _t(kernel)
        if delta.shape[1] != kernel_amount:
            raise B200Error(1, "the number of filters and the delta depth must match")
        if output_delta.shape[1] != kernel_z:
            raise B200Error(1, "wrong output depth for backward convolution")
        g = geom(kernel_z, output_delta.shape[2], output_delta.shape[3], kernel_amount, kernel_x, kernel_y, stride_x,
                 stride_y, padding_x, padding_y, delta.shape[2], delta.shape[3])
        _check(load().b200_conv_backward(C.byref(g), _ptr(output_delta), output_delta.shape[0], _ptr(delta), delta.shape[0],
                                         _ptr(kernel), kernel.shape[0], _ptr(bias) if bias is not None else None,
                                         bias.shape[0] if bias is not None else 0, _stream()))

    @staticmethod
    def _wgrad(fn, dkernel, kx, ky, kz, amount, dbias, image, delta, sx, sy, px, py, in_yx, out_yx):
        _t(dkernel), _t(dbias), _t(image), _t(delta)
        if dbias.shape[1] != amount:
            raise B200Error(1, "the number of kernel and bias corrections must match")
        g = geom(kz, in_yx[0], in_yx[1], amount, kx, ky, sx, sy, px, py, out_yx[0], out_yx[1])
        _check(fn(C.byref(g), _ptr(dkernel), dkernel.shape[0], _ptr(dbias), dbias.shape[0], _ptr(image), image.shape[0],
                  _ptr(delta), delta.shape[0], _stream()))

    @staticmethod
    def CreateDeltaWeightAndBias(dkernel, dkernel_x, dkernel_y, dkernel_z, dkernel_amount, dbias, image, delta,
                                 stride_x, stride_y, padding_x, padding_y):
        if image.shape[1] != dkernel_z or delta.shape[1] != dkernel_amount:
            raise B200Error(1, "image / delta depth does not match the kernel corrections")
        CTensorConv._wgrad(load().b200_conv_wgrad, dkernel, dkernel_x, dkernel_y, dkernel_z, dkernel_amount, dbias, image,
                           delta, stride_x, stride_y, padding_x, padding_y, image.shape[2:], delta.shape[2:])

    @staticmethod
    def CreateBackDeltaWeightAndBias(dkernel, dkernel_x, dkernel_y, dkernel_z, dkernel_amount, dbias, image, delta,
                                     stride_x, stride_y, padding_x, padding_y):
        if image.shape[1] != dkernel_amount or delta.shape[1] != dkernel_z:
            raise B200Error(1, "image / delta depth does not match the kernel corrections")
        CTensorConv._wgrad(load().b200_conv_back_wgrad, dkernel, dkernel_x, dkernel_y, dkernel_z, dkernel_amount, dbias,
                           image, delta, stride_x, stride_y, padding_x, padding_y, delta.shape[2:], image.shape[2:])

    @staticmethod
    def CreateDeltaWeightAndBiasBatch(dkernel, dkernel_x, dkernel_y, dkernel_z, dkernel_amount, dbias, image, delta,
                                      stride_x, stride_y, padding_x, padding_y, accumulate=True):
        """Batch-summed form used by the layers: dkernel [1,1,K,C*ky*kx] (+)= sum over the batch."""
        _t(dkernel), _t(image), _t(delta)
        g = geom(dkernel_z, image.shape[2], image.shape[3], dkernel_amount, dkernel_x, dkernel_y, stride_x, stride_y,
                 padding_x, padding_y, delta.shape[2], delta.shape[3])
        if image.shape[0] != delta.shape[0]:
            raise B200Error(1, "image and delta batch sizes differ")
        _check(load().b200_conv_wgrad_batch(C.byref(g), _ptr(dkernel), _ptr(dbias) if dbias is not None else None,
                                            int(accumulate), _ptr(image), _ptr(delta), image.shape[0], _stream()))


def _n(x):
    return x.shape[1] * x.shape[2] * x.shape[3]


def _same_zyx(*ts):
    s = ts[0].shape[1:]
    if any(t.shape[1:] != s for t in ts):
        raise B200Error(1, "tensor sizes do not match")


class CTensorMath:
    """cuda/ctensormath.cu.h:92-135."""

    @staticmethod
    def Mul(output, left, right, tensor_core=False):
        _t(output), _t(left), _t(right)
        if left.shape[3] != right.shape[2] or left.shape[1] != right.shape[1] or output.shape[2] != left.shape[2] or \
                output.shape[3] != right.shape[3] or output.shape[1] != right.shape[1]:
            raise B200Error(1, "CTensor::Mul: tensor sizes do not match")
        _check(load().b200_mul(_ptr(output), output.shape[0], _ptr(left), left.shape[0], _ptr(right), right.shape[0],
                               left.shape[1], left.shape[2], left.shape[3], right.shape[3], 0, _stream()))

    @staticmethod
    def TransponseMul(output, left, right, tensor_core=False):
        _t(output), _t(left), _t(right)
        if left.shape[2] != right.shape[2] or left.shape[1] != right.shape[1] or output.shape[2] != left.shape[3] or \
                output.shape[3] != right.shape[3] or output.shape[1] != right.shape[1]:
            raise B200Error(1, "CTensor::TransponseMul: tensor sizes do not match")
        _check(load().b200_mul(_ptr(output), output.shape[0], _ptr(left), left.shape[0], _ptr(right), right.shape[0],
                               left.shape[1], left.shape[2], left.shape[3], right.shape[3], 1, _stream()))

    @staticmethod
    def MulValue(output, inp, value):
        _t(output), _t(inp)
        _same_zyx(output, inp)
        _check(load().b200_unary(_ptr(output), output.shape[0], _ptr(inp), inp.shape[0], _n(output), 3, value, 0.0, _stream()))

    @staticmethod
    def Add(output, left, right, left_scale=1.0, right_scale=1.0):
        _t(output), _t(left), _t(right)
        _same_zyx(output, left, right)
        _check(load().b200_add(_ptr(output), output.shape[0], _ptr(left), left.shape[0], _ptr(right), right.shape[0],
                               _n(output), left_scale, right_scale, 0, _stream()))

    @staticmethod
    def Sub(output, left, right, left_scale=1.0, right_scale=1.0):
        _t(output), _t(left), _t(right)
        _same_zyx(output, left, right)
        _check(load().b200_add(_ptr(output), output.shape[0], _ptr(left), left.shape[0], _ptr(right), right.shape[0],
                               _n(output), left_scale, right_scale, 1, _stream()))

    @staticmethod
    def AddSumW(output, left, right, left_scale=1.0, right_scale=1.0):
        _t(output), _t(left), _t(right)
        _same_zyx(output, left, right)
        _check(load().b200_add_sum_w(_ptr(output), output.shape[0], _ptr(left), left.shape[0], _ptr(right), right.shape[0],
                                     _n(output), left_scale, right_scale, _stream()))

    @staticmethod
    def AddBias(working, bias):
        _t(working), _t(bias)
        if working.shape[1] != bias.shape[1]:
            raise B200Error(1, "CTensor::AddBias: tensor sizes do not match")
        _check(load().b200_add_bias(_ptr(working), working.shape[0], working.shape[1], working.shape[2] * working.shape[3],
                                    _ptr(bias), bias.shape[0], _stream()))

    @staticmethod
    def SummXY(output, inp):
        _t(output), _t(inp)
        if output.shape[1] != inp.shape[1]:
            raise B200Error(1, "CTensor::SummXY: tensor sizes do not match")
        _check(load().b200_summ_xy(_ptr(output), output.shape[0], _ptr(inp), inp.shape[0], inp.shape[1],
                                   inp.shape[2] * inp.shape[3], _stream()))

    @staticmethod
    def _unary(op, output, inp, a, b):
        _t(output), _t(inp)
        _same_zyx(output, inp)
        _check(load().b200_unary(_ptr(output), output.shape[0], _ptr(inp), inp.shape[0], _n(output), op, a, b, _stream()))

    @staticmethod
    def Pow2(output, inp, scale=1.0):
        CTensorMath._unary(0, output, inp, scale, 0.0)

    @staticmethod
    def SQRT(output, inp, scale, add_sqrt_value):
        CTensorMath._unary(1, output, inp, scale, add_sqrt_value)

    @staticmethod
    def Inv(output, inp):
        CTensorMath._unary(2, output, inp, 0.0, 0.0)

    @staticmethod
    def Set(output, inp, scale=1.0, add_value=0.0):
        """output = input*scale + add_value (cuda/ctensormath.cu.h: Set, AddValue, SubValue)."""
        CTensorMath._unary(4, output, inp, scale, add_value)

    @staticmethod
    def Clip(tensor, min_value, max_value):
        CTensorMath._unary(5, tensor, tensor, min_value, max_value)

    @staticmethod
    def Signum(tensor):
        CTensorMath._unary(6, tensor, tensor, 0.0, 0.0)

    @staticmethod
    def Div(output, left, right, left_scale=1.0, right_scale=1.0):
        """output = (left*left_scale) / (right*right_scale), W broadcast per operand."""
        _t(output), _t(left), _t(right)
        _same_zyx(output, left, right)
        _check(load().b200_div(_ptr(output), output.shape[0], _ptr(left), left.shape[0], _ptr(right), right.shape[0],
                               _n(output), left_scale, right_scale, _stream()))

    @staticmethod
    def Transponse(output, inp):
        """Every (w,z) plane transposed: output is [W,Z,X,Y] for an input [W,Z,Y,X]."""
        _t(output), _t(inp)
        if output.shape[0] != inp.shape[0] or output.shape[1] != inp.shape[1] or output.shape[2] != inp.shape[3] or output.shape[3] != inp.shape[2]:
            raise B200Error("CTensorMath::Transponse: tensor sizes do not match!")
        _check(load().b200_transpose(_ptr(output), _ptr(inp), inp.shape[0] * inp.shape[1], inp.shape[2], inp.shape[3], _stream()))

    @staticmethod
    def ConcatecationZ(output, input_a, input_b):
        _t(output), _t(input_a), _t(input_b)
        if output.shape[2:] != input_a.shape[2:] or output.shape[2:] != input_b.shape[2:] or \
                output.shape[1] != input_a.shape[1] + input_b.shape[1]:
            raise B200Error(1, "CTensor::ConcatecationZ: tensor sizes do not match")
        _check(load().b200_concat_z(_ptr(output), output.shape[0], _ptr(input_a), input_a.shape[0], input_a.shape[1], _ptr(input_b),
                                    input_b.shape[0], input_b.shape[1], output.shape[2] * output.shape[3], _stream()))

    @staticmethod
    def SplitZ(output_a, output_b, inp):
        _t(output_a), _t(output_b), _t(inp)
        if inp.shape[2:] != output_a.shape[2:] or inp.shape[2:] != output_b.shape[2:] or inp.shape[0] != output_a.shape[0] or \
                inp.shape[0] != output_b.shape[0] or inp.shape[1] != output_a.shape[1] + output_b.shape[1]:
            raise B200Error(1, "CTensor::SplitZ: tensor sizes do not match")
        _check(load().b200_split_z(_ptr(output_a), output_a.shape[1], _ptr(output_b), output_b.shape[1], _ptr(inp), inp.shape[0],
                                   inp.shape[2] * inp.shape[3], _stream()))

    @staticmethod
    def SetTimeStep(output, inp, time_step):
        """time_step: uint32 (torch.int32 storage) tensor [W,1,1,1] (cuda/ctensormath.cu.h:3061)."""
        _t(output), _t(inp)
        if output.shape != inp.shape or time_step.numel() != inp.shape[0] or time_step.dtype != torch.int32:
            raise B200Error(1, "CTensor::SetTimeStep: tensor sizes do not match")
        _check(load().b200_set_time_step(_ptr(output), _ptr(inp), _ptr(time_step), inp.shape[0], _n(inp), _stream()))

    @staticmethod
    def SetNormalNoise(output, seed):
        _t(output)
        _check(load().b200_normal_noise(_ptr(output), output.numel(), seed, _stream()))

    @staticmethod
    def CreateDropOutMatrix(output, drop_out, seed):
        _t(output)
        _check(load().b200_dropout_mask(_ptr(output), output.numel(), drop_out, seed, _stream()))

    @staticmethod
    def GetNoiseImageAndNoise(noisy_image, noise, image, sqrt_alpha_bar, sqrt_one_minus_alpha_bar, seed=None):
        """seed given: the noise is drawn and written to `noise` (the reference's behaviour, cuda/ctensormath.cu.h:3250);
        seed None: `noise` is an input supplied by the caller."""
        _t(noisy_image), _t(noise), _t(image), _t(sqrt_alpha_bar), _t(sqrt_one_minus_alpha_bar)
        if noisy_image.shape != noise.shape or noisy_image.shape != image.shape:
            raise B200Error(1, "CTensor::GetNoiseImageAndNoise: the sizes of NoisyImage, Noise and Image do not match")
        if sqrt_alpha_bar.numel() != image.shape[0] or sqrt_one_minus_alpha_bar.numel() != image.shape[0]:
            raise B200Error(1, "CTensor::GetNoiseImageAndNoise: the sizes of SqrtAlphaBar/SqrtOneMinusAlphaBar and Image do not match")
        _check(load().b200_noisy_image(_ptr(noisy_image), _ptr(noise), _ptr(image), _ptr(sqrt_alpha_bar), _ptr(sqrt_one_minus_alpha_bar),
                                       image.shape[0], _n(image), int(seed is not None), seed or 0, _stream()))

    @staticmethod
    def TensorItemProduction(output, left, right):
        _t(output), _t(left), _t(right)
        _same_zyx(output, left, right)
        _check(load().b200_item_product(_ptr(output), output.shape[0], _ptr(left), left.shape[0], _ptr(right),
                                        right.shape[0], _n(output), _stream()))

    @staticmethod
    def Fill(output, value=0.0):
        _t(output)
        _check(load().b200_fill(_ptr(output), output.numel(), value, _stream()))

    @staticmethod
    def MaxPooling(output, position, inp, pooling_x, pooling_y):
        _t(output), _t(inp)
        if inp.shape[3] // pooling_x != output.shape[3] or inp.shape[2] // pooling_y != output.shape[2] or \
                inp.shape[:2] != output.shape[:2]:
            raise B200Error(1, "CTensor::MaxPooling: tensor sizes do not match")
        _check(load().b200_maxpool(_ptr(output), _ptr(position), _ptr(inp), inp.shape[0], inp.shape[1], inp.shape[2],
                                   inp.shape[3], pooling_x, pooling_y, _stream()))

    @staticmethod
    def MaxPoolingBackward(output, position, inp, pooling_x, pooling_y):
        _t(output), _t(inp)
        if inp.shape[3] != output.shape[3] // pooling_x or inp.shape[2] != output.shape[2] // pooling_y or \
                inp.shape[:2] != output.shape[:2]:
            raise B200Error(1, "CTensor::MaxPooling: tensor sizes do not match")
        _check(load().b200_maxpool_backward(_ptr(output), _ptr(position), _ptr(inp), output.shape[0], output.shape[1],
                                            output.shape[2], output.shape[3], pooling_x, pooling_y, _stream()))

    @staticmethod
    def UpSampling(output, inp, upsampling_x, upsampling_y):
        _t(output), _t(inp)
        if inp.shape[3] != output.shape[3] // upsampling_x or inp.shape[2] != output.shape[2] // upsampling_y or \
                inp.shape[1] != output.shape[1]:
            raise B200Error(1, "CTensor::UpSampling: tensor sizes do not match")
        _check(load().b200_upsample(_ptr(output), _ptr(inp), inp.shape[0], inp.shape[1], inp.shape[2], inp.shape[3],
                                    upsampling_x, upsampling_y, _stream()))

    @staticmethod
    def DownSampling(output, inp, downsampling_x, downsampling_y):
        _t(output), _t(inp)
        if inp.shape[3] // downsampling_x != output.shape[3] or inp.shape[2] // downsampling_y != output.shape[2] or \
                inp.shape[:2] != output.shape[:2]:
            raise B200Error(1, "CTensor::DownSampling: tensor sizes do not match")
        _check(load().b200_downsample(_ptr(output), _ptr(inp), inp.shape[0], inp.shape[1], inp.shape[2], inp.shape[3],
                                      downsampling_x, downsampling_y, _stream()))

    @staticmethod
    def Adam(weight, dweight, m, v, batch_size, speed, beta1, beta2, epsilon, iteration):
        _t(weight), _t(dweight), _t(m), _t(v)
        if not (weight.shape == dweight.shape == m.shape == v.shape):
            raise B200Error(1, "CTensor::Adam: tensor sizes do not match")
        _check(load().b200_adam(_ptr(weight), _ptr(dweight), _ptr(m), _ptr(v), weight.numel(), batch_size, speed, beta1,
                                beta2, epsilon, iteration, _stream()))


class CTensorApplyFunc:
    """cuda/ctensorapplyfunc.cu.h:78-90; `func` is one of ACT."""

    @staticmethod
    def Apply(output, inp, func, leaky_slope=0.1):
        _t(output), _t(inp)
        _check(load().b200_activation(_ptr(output), _ptr(inp), inp.numel(), ACT[func], 0, leaky_slope, _stream()))

    @staticmethod
    def ApplyDifferential(output, inp, func, leaky_slope=0.1):
        _t(output), _t(inp)
        _check(load().b200_activation(_ptr(output), _ptr(inp), inp.numel(), ACT[func], 1, leaky_slope, _stream()))

    @staticmethod
    def Backward(output, z, error, func, leaky_slope=0.1):
        """output = f'(z) * error.  z may be a Checkpoint8 (of the function's input); output and error then may be fp32, bf16 or fp16."""
        if isinstance(z, Checkpoint8):
            dev = _device()
            kind, rows, n, pitch = z._match(output, "output", dev)
            error_pitch = _like(error, "error", (kind, rows, n), "output", dev)
            _check(load().b200_ckpt8_activation_backward(output.data_ptr(), z.codes.data_ptr(), z.exponents.data_ptr(), error.data_ptr(),
                                                         kind, rows, n, pitch, error_pitch, ACT[func], leaky_slope, _raw_stream(dev)))
            return
        _t(output), _t(z), _t(error)
        _check(load().b200_activation_backward(_ptr(output), _ptr(z), _ptr(error), z.numel(), ACT[func], leaky_slope, _stream()))

    @staticmethod
    def BiasActivation(working, bias, func, leaky_slope=0.1, pre=None):
        _t(working), _t(bias)
        _check(load().b200_bias_activation(_ptr(working), _ptr(pre) if pre is not None else None, working.shape[0],
                                           working.shape[1], working.shape[2] * working.shape[3], _ptr(bias), ACT[func],
                                           leaky_slope, _stream()))


def bn_forward(x, gamma, beta, momentum=0.9, eps=1e-6, new_mean=None, new_var=None):
    """CNetLayerBatchNormalization::Forward (training).  Returns dict(y, xhat, ivar, mean, var)."""
    _t(x), _t(gamma), _t(beta)
    y, xhat = torch.empty_like(x), torch.empty_like(x)
    ivar, mean, var = (torch.empty_like(gamma) for _ in range(3))
    _check(load().b200_bn_forward(_ptr(y), _ptr(xhat), _ptr(ivar), _ptr(mean), _ptr(var),
                                  _ptr(new_mean) if new_mean is not None else None,
                                  _ptr(new_var) if new_var is not None else None, _ptr(x), _ptr(gamma), _ptr(beta),
                                  x.shape[0], x[0].numel(), momentum, eps, _stream()))
    return dict(y=y, xhat=xhat, ivar=ivar, mean=mean, var=var)


def bn_backward(dy, xhat, ivar, gamma, dgamma, dbeta, create_delta_weight=True):
    _t(dy), _t(xhat), _t(ivar), _t(gamma)
    dx = torch.empty_like(dy)
    _check(load().b200_bn_backward(_ptr(dx), _ptr(dgamma), _ptr(dbeta), _ptr(dy), _ptr(xhat), _ptr(ivar), _ptr(gamma),
                                   dy.shape[0], dy[0].numel(), int(create_delta_weight), _stream()))
    return dx


def _workspace(size, given, name, like, dev):
    """(tensor, address, bytes) of the caller's workspace, or of a fresh one from torch's allocator (which orders its reuse by stream
    and keeps the workspaces of captured graphs apart); `like`: an fp32 tensor on the current device."""
    if given is None:
        if not size:
            return None, None, 0
        given = like.new_empty((size + 3) // 4)
        return given, given.data_ptr(), size
    if not (isinstance(given, torch.Tensor) and given.is_cuda and given.is_contiguous() and given.get_device() == dev):
        raise B200Error(2, f"{name}: the workspace must be a contiguous tensor on the current device")
    return given, given.data_ptr(), given.numel() * given.element_size()


def ln_forward(x, gamma, beta, eps=1e-6, y=None, mean=None, rstd=None, checkpoint=None):
    """Layer normalisation of every row of x (its first dimension is the rows, the others are normalised together) in fp32,
    bf16 or fp16 with fp32 parameters.  checkpoint: a Checkpoint8 that receives the normalised values for ln_backward.
    Returns dict(y, mean, rstd)."""
    dev = _device()
    kind, rows, n, pitch = _rows(x, "x", dev)
    if y is None:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if mean is None:
        mean = torch.empty(rows, device=x.device)
    if rstd is None:
        rstd = torch.empty(rows, device=x.device)
    y_pitch = _like(y, "y", (kind, rows, n), "x", dev)
    codes = exponents = None
    if checkpoint is not None:
        if checkpoint._here(dev).rows != rows or checkpoint.n != n:
            raise B200Error(1, f"the checkpoint must have {rows} rows of {n} values")
        codes, exponents = checkpoint.codes.data_ptr(), checkpoint.exponents.data_ptr()
    _check(load().b200_ln_forward(y.data_ptr(), _param(mean, rows, "mean", dev), _param(rstd, rows, "rstd", dev), codes, exponents,
                                  x.data_ptr(), _param(gamma, n, "gamma", dev), _param(beta, n, "beta", dev), kind, rows, n, pitch,
                                  y_pitch, eps, _raw_stream(dev)))
    return dict(y=y, mean=mean, rstd=rstd)


def ln_backward(dy, x, mean, rstd, gamma, dgamma, dbeta, create_delta_weight=True, accumulate=True, dx=None, workspace=None):
    """Backward pass of ln_forward; returns dx.  x: the input of the forward pass, or the Checkpoint8 it filled (mean is then
    not read and may be None).  dgamma, dbeta (fp32, n elements) are added to, or written with accumulate=False."""
    dev = _device()
    kind, rows, n, dy_pitch = _rows(dy, "dy", dev)
    if dx is None:
        dx = torch.empty(dy.shape, dtype=dy.dtype, device=dy.device)
    dx_pitch = _like(dx, "dx", (kind, rows, n), "dy", dev)
    codes = exponents = x_ptr = mean_ptr = dg = db = None
    x_pitch = n
    if isinstance(x, Checkpoint8):
        if x._here(dev).rows != rows or x.n != n:
            raise B200Error(1, f"the checkpoint must have {rows} rows of {n} values")
        codes, exponents = x.codes.data_ptr(), x.exponents.data_ptr()
    else:
        x_pitch = _like(x, "x", (kind, rows, n), "dy", dev)
        x_ptr, mean_ptr = x.data_ptr(), _param(mean, rows, "mean", dev)
    gamma_ptr, rstd_ptr = _param(gamma, n, "gamma", dev), _param(rstd, rows, "rstd", dev)
    if create_delta_weight:
        dg, db = _param(dgamma, n, "dgamma", dev), _param(dbeta, n, "dbeta", dev)
    lib = load()
    workspace, ws, size = _workspace(lib.b200_ln_backward_workspace(rows, n), workspace, "ln_backward", gamma, dev)
    _check(lib.b200_ln_backward(dx.data_ptr(), dg, db, dy.data_ptr(), x_ptr, mean_ptr, rstd_ptr, codes, exponents, gamma_ptr,
                                kind, rows, n, dx_pitch, dy_pitch, x_pitch, int(create_delta_weight), int(accumulate), ws, size,
                                _raw_stream(dev)))
    return dx


def checkpoint_wgrad(dweight, dbias, delta, checkpoint, accumulate=True, workspace=None):
    """Gradients of a Linear layer whose input was kept in 8 bits: dweight [out x n] (+)= delta^T * values and, unless dbias is
    None, dbias [out] (+)= sum of delta over the rows.  delta [rows x out] in fp32, bf16 or fp16; the gradients are fp32."""
    dev = _device()
    kind, rows, out, pitch = _rows(delta, "delta", dev)
    n = checkpoint.n
    if checkpoint._here(dev).rows != rows:
        raise B200Error(1, "delta and the checkpoint must have the same number of rows")
    dw, db, d = _param(dweight, out * n, "dweight", dev), None if dbias is None else _param(dbias, out, "dbias", dev), delta.data_ptr()
    lib = load()
    workspace, ws, size = _workspace(lib.b200_ckpt8_wgrad_workspace(kind, rows, out, n, d, pitch), workspace, "checkpoint_wgrad", dweight, dev)
    _check(lib.b200_ckpt8_wgrad(dw, db, int(accumulate), d, checkpoint.codes.data_ptr(), checkpoint.exponents.data_ptr(), kind, rows, out,
                                n, pitch, ws, size, _raw_stream(dev)))


def vae_forward(mu, logvar, eps, want_kl=True):
    _t(mu), _t(logvar), _t(eps)
    z = torch.empty_like(mu)
    kl = C.c_float(0.0)
    _check(load().b200_vae_forward(_ptr(z), _ptr(mu), _ptr(logvar), _ptr(eps), mu.shape[0], mu[0].numel(),
                                   C.byref(kl) if want_kl else None, _stream()))
    return z, kl.value


def vae_backward(delta, mu, logvar, eps, kl_speed):
    _t(delta), _t(mu), _t(logvar), _t(eps)
    dmu, dlv = torch.empty_like(mu), torch.empty_like(mu)
    _check(load().b200_vae_backward(_ptr(dmu), _ptr(dlv), _ptr(delta), _ptr(mu), _ptr(logvar), _ptr(eps), mu.numel(),
                                    kl_speed, _stream()))
    return dmu, dlv


def prepack_conv_layers(layers, kernels):
    """b200_conv_layers_prepack: the tensor-core weight packs of several ConvLayer objects in one launch, each good for the
    layer's next forward call with that kernel tensor."""
    if not layers:
        return
    handles = (C.c_void_p * len(layers))(*[layer._h for layer in layers])
    pointers = (C.c_void_p * len(layers))(*[_t(k).data_ptr() for k in kernels])
    _check(load().b200_conv_layers_prepack(handles, pointers, len(layers), _stream()))


class ConvLayer:
    """Forward / TrainingBackward of the reference's convolution layer (netlayer/cnetlayerconvolution.cu.h:310,484)
    or, with transposed=True, of its transposed-convolution layer (netlayer/cnetlayerbackconvolution.cu.h:303,475).
    The library context keeps the packed layer input between the two calls."""

    def __init__(self, in_z, in_y, in_x, kernel_amount, kernel_x, kernel_y, stride_x, stride_y, padding_x, padding_y, batch,
                 transposed=False):
        self.g = geom(in_z, in_y, in_x, kernel_amount, kernel_x, kernel_y, stride_x, stride_y, padding_x, padding_y)
        self.batch, self.transposed = batch, transposed
        self._h = C.c_void_p()
        _check(load().b200_conv_layer_create(C.byref(self._h), C.byref(self.g), batch, int(transposed)))

    def forward(self, output, inp, kernel, bias=None):
        _t(output), _t(inp), _t(kernel)
        _check(load().b200_conv_layer_forward(self._h, _ptr(output), _ptr(inp), _ptr(kernel),
                                              _ptr(bias) if bias is not None else None, _stream()))

    def forward_fused(self, output, inp, kernel, bias=None, input_func=None, input_slope=0.1, input_act_out=None, output_func=None,
                      output_slope=0.1, output_pre=None):
        """b200_conv_layer_forward_fused: input_func is the function layer in front of this layer (applied while the input is
        packed; input_act_out optionally receives f(inp)), output_func the one behind it (applied in the epilogue; output_pre
        optionally receives the value before the function)."""
        from .lib import ConvFusion
        _t(output), _t(inp), _t(kernel)
        f = ConvFusion(ACT[input_func] if input_func else -1, input_slope, input_act_out.data_ptr() if input_act_out is not None else None,
                       ACT[output_func] if output_func else -1, output_slope, output_pre.data_ptr() if output_pre is not None else None)
        _check(load().b200_conv_layer_forward_fused(self._h, _ptr(output), _ptr(inp), _ptr(kernel), _ptr(bias) if bias is not None else None,
                                                    C.byref(f), _stream()))

    def backward(self, input_delta, dkernel, dbias, output_delta, inp, kernel, accumulate=True):
        _t(output_delta), _t(inp), _t(kernel)
        _check(load().b200_conv_layer_backward(self._h, _ptr(input_delta) if input_delta is not None else None,
                                               _ptr(dkernel) if dkernel is not None else None,
                                               _ptr(dbias) if dbias is not None else None, int(accumulate),
                                               _ptr(output_delta), _ptr(inp), _ptr(kernel), _stream()))

    def forget_error(self):
        """The next backward call packs its output error anew, even if it is the tensor of the weights-only call before it."""
        _check(load().b200_conv_layer_forget_error(self._h))

    def close(self):
        if self._h:
            load().b200_conv_layer_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
