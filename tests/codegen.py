"""The machine code of a library built here: its kernels' instructions, from the code objects in it."""
import os
import re
import struct
import subprocess

BIN = "/opt/rocm/llvm/bin"


def tools():
    return all(os.path.exists(os.path.join(BIN, t)) for t in ("llvm-objcopy", "llvm-objdump"))


def code_objects(lib, folder):
    """The gfx950 code objects of a library, as files."""
    dump = os.path.join(folder, "fatbin")
    subprocess.check_call([BIN + "/llvm-objcopy", "--dump-section", ".hip_fatbin=" + dump, lib, os.devnull])
    data, files = open(dump, "rb").read(), []
    for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", data):
        at = m.end() + 8
        for _ in range(struct.unpack_from("<Q", data, m.end())[0]):
            start, size, n = struct.unpack_from("<QQQ", data, at)
            target = data[at + 24:at + 24 + n]
            at += 24 + n
            if b"gfx950" in target:
                files.append(os.path.join(folder, "co%d" % len(files)))
                with open(files[-1], "wb") as f:
                    f.write(data[m.start() + start:m.start() + start + size])
    return files


def disassembly(code_object):
    """The path of a listing: `<symbol>:`, `<L3>:` and instructions."""
    out = code_object + ".s"
    with open(out, "w") as f:
        subprocess.check_call([BIN + "/llvm-objdump", "-d", "--no-show-raw-insn", "--no-leading-addr", "--symbolize-operands", code_object], stdout=f)
    return out


def kernels(listing):
    """(symbol, its instructions and labels as texts) of each function."""
    name, body = None, []
    with open(listing) as f:
        for line in f:
            text = line.split("//")[0].strip()
            if not text:
                continue
            if text[0] == "<" and text[-2:] == ">:":
                label = text[1:-2]
                if re.match(r"L\d+$", label):
                    body.append(label + ":")
                else:
                    if name:
                        yield name, body
                    name, body = label, []
            elif name:
                body.append(text)
    if name:
        yield name, body


_LANES = ("v_", "ds_", "buffer_", "global_", "flat_", "scratch_")
_EXEC = re.compile(r"s_(cbranch|branch|endpgm|setpc|swappc|\w*saveexec|\w+ exec[,_ ])")


def before_the_lanes_are_back(body):
    """Vector instructions between a label that a branch on empty lanes goes to and the s_or_b64 that turns those lanes on again: a
    wave that took the branch runs them with no lane on, and they do nothing.  What a later instruction needs of them for all
    lanes (a register saved there) is then lost."""
    targets = {text.split()[1] for text in body if text.startswith("s_cbranch_execz ")}
    found = []
    for i, text in enumerate(body):
        if not text.endswith(":") or text[:-1] not in targets:
            continue
        seen = []
        for t in body[i + 1:]:
            if t.startswith("s_or_b64 exec, exec,"):
                found += [(text[:-1], s) for s in seen]
                break
            if t.endswith(":") or _EXEC.match(t):
                break
            if t.startswith(_LANES) and "readlane" not in t and "writelane" not in t:
                seen.append(t)
    return found
