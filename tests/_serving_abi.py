"""ctypes view of the batched serving operators' C ABI, made from include/vtq.h itself."""
import ctypes
import os
import re

from vtq import load_library

_SRC = re.sub(r"/\*.*?\*/", "", open(os.path.join(os.path.dirname(__file__), "..", "include", "vtq.h")).read(), flags=re.S)
_TYPES = {"int64_t": ctypes.c_int64, "int32_t": ctypes.c_int32, "uint32_t": ctypes.c_uint32, "float": ctypes.c_float,
          "size_t": ctypes.c_size_t, "vtq_status": ctypes.c_int32}


def struct(name):
    """The structure `name` of the header; fields by the header's names."""
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), _SRC, flags=re.S).group(1)
    fields = []
    for decl in body.split(";"):
        m = re.match(r"(?:const )?(\w+)\s*(.*)", decl.strip(), flags=re.S)
        if not m or not m.group(2):
            continue
        for field in m.group(2).split(","):
            field = field.strip()
            fields.append((field.lstrip("* "), ctypes.c_void_p if "*" in field else _TYPES[m.group(1)]))
    cls = type(name, (ctypes.Structure,), {"_fields_": fields})
    _TYPES[name] = cls
    return cls


def function(name):
    """The entry point `name` with the header's argument types."""
    res, args = re.search(r"(\w+\*?) %s\((.*?)\);" % name, _SRC, flags=re.S).groups()
    fn = getattr(load_library(), name)
    fn.restype = _TYPES[res]
    fn.argtypes = [ctypes.c_void_p if "*" in a else _TYPES[re.sub(r"^const ", "", a.strip()).split()[0]] for a in args.split(",")]
    return fn


def last_error():
    fn = load_library().vtq_device_last_error
    fn.restype = ctypes.c_char_p
    return fn().decode()


LinearI8, PagedKV, AppendKV, Attention, Verify = (struct("vtq_" + n) for n in (
    "linear_i8_args", "paged_kv", "append_kv_args", "attention_args", "verify_args"))
F32, F16, I8, BF16 = (int(re.search(r"#define VTQ_%s (\d+)" % n, _SRC).group(1)) for n in ("F32", "F16", "I8", "BF16"))
